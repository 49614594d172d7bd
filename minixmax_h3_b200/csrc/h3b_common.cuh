// Shared device helpers for the sm_100a kernels of the DiT-block hot path:
// status words, bounded mbarrier waits, TMA (non-multicast) copies, tcgen05
// (TMEM alloc / MMA / ld / st / cp / commit) wrappers and UMMA descriptors.
//
// Every spin in this library is bounded: a wait that exceeds its time budget
// records an error in the translation unit's device status word, raises the
// CTA-local abort flag and returns false, so the kernel unwinds instead of
// hanging the GPU.  No helper here issues a multicast load.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/h3b.h"

#define H3B_DEV __device__ __forceinline__

// ----------------------------------------------------------------------------
// Status words.  Each translation unit owns one `g_status` (code, site, info,
// block) in device memory; the host reads it through the registry in abi.cpp.
// ----------------------------------------------------------------------------
struct H3bDeviceStatus {
  int code;
  int site;
  int info;
  int block;
};

#define H3B_DECLARE_STATUS() static __device__ H3bDeviceStatus g_status = {0, 0, 0, 0}

// Bounded-wait budget in nanoseconds of %globaltimer (about two seconds).  A
// healthy pipeline wait lasts microseconds; reaching this means a deadlock.
#define H3B_WAIT_NS (2000ull * 1000ull * 1000ull)

H3B_DEV uint64_t globaltimer_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

H3B_DEV uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

H3B_DEV bool elect_one() {
  uint32_t pred = 0;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "elect.sync _|P, 0xffffffff;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(pred));
  return pred != 0;
}

// ----------------------------------------------------------------------------
// mbarrier
// ----------------------------------------------------------------------------
H3B_DEV void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}

H3B_DEV void fence_barrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

H3B_DEV void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

H3B_DEV void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

// try_wait with an explicit suspend-time hint (ns): the thread sleeps until
// the phase completes or the hint expires, whichever comes first.
H3B_DEV bool mbar_try_wait(uint32_t bar_addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 P, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar_addr), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}

// try_wait without a suspend hint: polls without yielding, for a thread whose
// reaction time is on the critical path (a single MMA-issuing thread).
H3B_DEV bool mbar_try_wait_spin(uint32_t bar_addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar_addr), "r"(parity)
      : "memory");
  return ok != 0;
}

// Cluster-scope acquire: for a barrier that threads of the other CTA of a
// cluster arrive on (their release.cluster arrivals pair with it).
H3B_DEV bool mbar_try_wait_cluster(uint32_t bar_addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar_addr), "r"(parity)
      : "memory");
  return ok != 0;
}

// Out-of-line part of a compact wait: `t0` 0 starts the clock; returns 0 when
// the wait is to be given up (budget spent, reported; or another warp of the
// CTA has given up), else the start time.
static __device__ __noinline__ uint64_t mbar_overdue(uint64_t t0, H3bDeviceStatus* st, int site, int parity,
                                                     volatile int* abort_flag) {
  if (abort_flag != nullptr && *abort_flag) return 0;
  const uint64_t now = globaltimer_ns();
  if (t0 == 0) return now;
  if (now - t0 <= H3B_WAIT_NS) return t0;
  if (atomicCAS(&st->code, 0, H3B_ERR_DEVICE_TIMEOUT) == 0) {
    st->site = site;
    st->info = parity;
    st->block = static_cast<int>(blockIdx.x);
  }
  if (abort_flag != nullptr) *abort_flag = 1;
  return 0;
}

// Wait for phase `parity` of `bar` to complete.  Returns false (and records
// `site` in *st, raising *abort_flag) when the budget runs out or when another
// warp of the CTA already aborted.  SPIN: poll without a suspend hint;
// CLUSTER: cluster-scope acquire (polls too).  COMPACT: the clock and the
// report stay out of line (~1 KB less code a wait, for kernels whose warps
// run different code from one instruction cache).
template <bool SPIN = false, bool CLUSTER = false, bool COMPACT = false>
H3B_DEV bool mbar_wait(uint64_t* bar, uint32_t parity, H3bDeviceStatus* st, int site,
                       volatile int* abort_flag) {
  const uint32_t addr = smem_u32(bar);
  auto poll = [&]() {
    return CLUSTER ? mbar_try_wait_cluster(addr, parity)
                   : (SPIN ? mbar_try_wait_spin(addr, parity) : mbar_try_wait(addr, parity));
  };
  if (poll()) return true;
  uint64_t t0 = COMPACT ? 0 : globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    if (poll()) return true;
    if ((++spins & 255u) == 0) {
      if constexpr (COMPACT) {
        t0 = mbar_overdue(t0, st, site, static_cast<int>(parity), abort_flag);
        if (t0 == 0) return false;
        continue;
      }
      if (abort_flag != nullptr && *abort_flag) return false;
      if (globaltimer_ns() - t0 > H3B_WAIT_NS) {
        if (atomicCAS(&st->code, 0, H3B_ERR_DEVICE_TIMEOUT) == 0) {
          st->site = site;
          st->info = static_cast<int>(parity);
          st->block = static_cast<int>(blockIdx.x);
        }
        if (abort_flag != nullptr) *abort_flag = 1;
        return false;
      }
    }
  }
}

// ----------------------------------------------------------------------------
// TMA (tensor and plain bulk copies, never multicast)
// ----------------------------------------------------------------------------
H3B_DEV void tma_load_2d(void* smem_dst, const CUtensorMap* map, int32_t x, int32_t y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

H3B_DEV void tma_load_3d(void* smem_dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z,
                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

H3B_DEV void tma_load_4d(void* smem_dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w,
                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}

// The tile into L2 only, ahead of its load.
H3B_DEV void tma_prefetch_4d(const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(z), "r"(w)
               : "memory");
}

H3B_DEV void bulk_load(void* smem_dst, const void* gmem_src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(smem_dst)),
      "l"(gmem_src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// TMA tensor store smem -> global (bulk-group completion), never a reduce.
// Stores clip at the tensor bounds; the caller never starts one at a negative
// coordinate.
H3B_DEV void tma_store_2d(const CUtensorMap* map, const void* smem_src, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_u32(smem_src))
               : "memory");
}
H3B_DEV void bulk_commit_group() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// Wait until at most N committed bulk groups still read shared memory.
template <int N>
H3B_DEV void bulk_wait_group_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
template <int N>
H3B_DEV void bulk_wait_group() {
  asm volatile("cp.async.bulk.wait_group %0;" ::"n"(N) : "memory");
}
// Make generic-proxy shared-memory writes visible to the async (TMA) proxy.
H3B_DEV void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

H3B_DEV void prefetch_tmap(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// ----------------------------------------------------------------------------
// tcgen05: TMEM allocation, fences, MMA, commit, ld/st/cp
// ----------------------------------------------------------------------------
H3B_DEV void tmem_alloc(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)),
               "r"(ncols)
               : "memory");
}
H3B_DEV void tmem_relinquish() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::); }
H3B_DEV void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
H3B_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
H3B_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
H3B_DEV void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
H3B_DEV void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Make the mbarrier track completion of every tcgen05 async op issued so far by
// this thread (MMA reads of smem included).
H3B_DEV void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T, kind::f16 (bf16 inputs, fp32 accumulate).
H3B_DEV void mma_f16_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// D[tmem] (+)= A[tmem] * B[smem], kind::f16 with the A operand in TMEM.
H3B_DEV void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// D[tmem] (+)= A[smem] * B[smem]^T, kind::i8 (s8 inputs, s32 accumulate).
H3B_DEV void mma_i8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Block-scaled NVFP4 MMA: e2m1 operands, one ue4m3 scale per 16 elements.
H3B_DEV void mma_nvf4_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa_tmem,
                         uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem));
}

// ----------------------------------------------------------------------------
// CTA pairs (cluster of 2, tcgen05 cta_group::2): the MMA of the leader CTA
// (cluster rank 0) reads its A rows and half of B from each CTA's shared
// memory at the same offsets and accumulates into each CTA's own TMEM.
// ----------------------------------------------------------------------------
H3B_DEV uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// shared::cluster address of the same shared-memory object in CTA `rank`.
H3B_DEV uint32_t mapa_shared(uint32_t cta_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(cta_addr), "r"(rank));
  return r;
}
// All threads of both CTAs.
H3B_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
H3B_DEV void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Arrive on the other CTA's mbarrier with the default semantics.  For a
// hand-off of TMEM contents the arriving warp has completed
// (tcgen05.wait::st / wait::ld, then tcgen05.fence::before_thread_sync),
// which the cluster-scope release above would only delay (~1000 cycles).
H3B_DEV void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// This CTA's share of a pair operand; the bytes complete on the leader's
// mbarrier (`leader_bar`, a shared::cluster address).  No multicast.
H3B_DEV void tma_load_2d_pair(void* smem_dst, const CUtensorMap* map, int32_t x, int32_t y, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}
H3B_DEV void tmem_alloc_pair(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_result)),
               "r"(ncols)
               : "memory");
}
H3B_DEV void tmem_relinquish_pair() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::); }
H3B_DEV void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// Commit the leader's pair MMAs to the mbarrier at this offset in every CTA of
// `cta_mask` (the commit's multicast; loads never multicast).
H3B_DEV void tc_commit_pair_mc(uint64_t* bar, uint16_t cta_mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(cta_mask)
      : "memory");
}
H3B_DEV void tc_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
H3B_DEV void mma_i8_ss_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}
// Block-scaled NVFP4 pair MMA: each CTA's scale operands are read from its
// own TMEM at the given columns.
H3B_DEV void mma_nvf4_ss_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa_tmem,
                              uint32_t sfb_tmem, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
          d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem));
}


// 32 lanes x 32 consecutive 32-bit columns -> 32 registers per thread.
H3B_DEV void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// tcgen05.ld writes its registers asynchronously: they are valid only after
// tcgen05.wait::ld.  The compiler does not know that, so after the wait the
// registers are passed through an empty volatile asm that "modifies" them;
// every later use then depends on a statement ordered after the wait.
H3B_DEV void reg_fence32(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// Load 32 columns into r[0..31] (pointer form of tmem_ld32).
H3B_DEV void tmem_ld32p(uint32_t taddr, uint32_t* r) { tmem_ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r)); }

H3B_DEV void reg_fence16(uint32_t* r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]));
}

// Wait for every outstanding tcgen05.ld of this thread and fence n*32 registers.
template <int N>
H3B_DEV void tmem_wait_fence(uint32_t* r) {
  tc_wait_ld();
#pragma unroll
  for (int c = 0; c < N; ++c) reg_fence32(r + 32 * c);
}

H3B_DEV void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

H3B_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

H3B_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// ----------------------------------------------------------------------------
// UMMA descriptors
// ----------------------------------------------------------------------------
// Shared-memory matrix descriptor, 128-byte swizzle, K-major operand: rows of
// 128 bytes, 8-row atoms 1024 bytes apart (SBO), LBO unused (encoded 1),
// version 1 (sm_100), layout type 2 (SWIZZLE_128B).  The tile base must be
// 1024-byte aligned; advancing K inside the atom adds bytes>>4 to the start.
H3B_DEV uint64_t sdesc_kmajor_sw128(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}

// MN-major operand with 128-byte swizzle: 64 bf16 along MN per 128-byte row,
// 8 K-rows per 1024-byte atom.  LBO = byte distance between 64-wide MN atoms,
// SBO = byte distance between consecutive 8-row K groups.
H3B_DEV uint64_t sdesc_mnmajor_sw128(uint32_t saddr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lbo_bytes >> 4) << 16) |
         (static_cast<uint64_t>(sbo_bytes >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// Advances a shared-memory descriptor by `delta` (bytes >> 4) in its start
// address field: one 32-bit add on the low word.  Valid while the resulting
// address stays inside the same operand allocation below 256 KB of shared
// memory, where the 14-bit field cannot carry into the next field.
H3B_DEV uint64_t desc_add_lo(uint64_t d, uint32_t delta) {
  const uint32_t lo = static_cast<uint32_t>(d) + delta;
  return (d & 0xFFFFFFFF00000000ull) | lo;
}

// Instruction descriptors (kind::f16 / kind::i8 share this format).
//  bits [4,6) D format (1 = f32, 2 = s32); [7,10) A format; [10,13) B format;
//  15 / 16 A / B major (0 = K, 1 = MN); [17,23) N>>3; [24,29) M>>4.
__host__ __device__ constexpr uint32_t idesc_bf16_f32(uint32_t m, uint32_t n, uint32_t a_mn_major,
                                                      uint32_t b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn_major << 15) | (b_mn_major << 16) | ((n >> 3) << 17) |
         ((m >> 4) << 24);
}
__host__ __device__ constexpr uint32_t idesc_f16_f32(uint32_t m, uint32_t n, uint32_t a_mn_major,
                                                     uint32_t b_mn_major) {
  return (1u << 4) | (a_mn_major << 15) | (b_mn_major << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__host__ __device__ constexpr uint32_t idesc_s8_s32(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// Block-scaled kind::mxf4nvf4: A/B format 1 (e2m1), scale format 0 (ue4m3),
// scale-factor ids 0, K = 64 per instruction.
__host__ __device__ constexpr uint32_t idesc_nvf4(uint32_t m, uint32_t n) {
  return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// ----------------------------------------------------------------------------
// Small numeric helpers
// ----------------------------------------------------------------------------
// fp32 -> nearest-even bf16 -> fp32 (one rounding step of a bf16 computation).
H3B_DEV float bf16r(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }

// Exact-erf GELU in fp32 (torch.nn.functional.gelu, approximate="none").
H3B_DEV float gelu_erf(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f)); }

// max |bf16(gelu(y))| over y < 0 is bf16(gelu(-0.7518..)) = -0.169921875 in
// magnitude: GELU's minimum is -0.16997, which rounds to 174 * 2^-10.
constexpr float GELU_BF16_NEG_BOUND = 0.169921875f;

// Global max |u| of u = bf16(gelu(y)) over bf16 values y, from
//   ymax2[0] = max(0, max y)   (GELU and bf16 rounding are monotone on y >= 0)
//   ymax2[1] = max |bf16(gelu(y))| by a full scan, needed (and present) only
//              when bf16(gelu(ymax2[0])) is below the bound for y < 0.
H3B_DEV float gelu_input_amax(const float* ymax2) {
  const float a = bf16r(gelu_erf(ymax2[0]));
  return a >= GELU_BF16_NEG_BOUND ? a : ymax2[1];
}
// The same rounding for two values with one packed conversion.
H3B_DEV float2 bf16r2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  const uint32_t u = *reinterpret_cast<const uint32_t*>(&h);
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
H3B_DEV float bf16lo_to_f32(uint32_t v) { return __uint_as_float(v << 16); }
H3B_DEV float bf16hi_to_f32(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }

H3B_DEV uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

H3B_DEV uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool F16>
H3B_DEV uint32_t pack16x2(float lo, float hi) {
  return F16 ? pack_f16x2(lo, hi) : pack_bf16x2(lo, hi);
}

// One 32-byte global store (sm_100 256-bit vector store).  The address must
// be 32-byte aligned.  Over NVLink a 32-byte granule written whole costs its
// own bytes; a 16-byte store costs a full granule.
H3B_DEV void st_global_v8(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// Packed fp32x2 arithmetic (sm_100): two lanes of work per instruction.
H3B_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)),
        "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
H3B_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
// Two round-to-nearest sums, bit-identical to two __fadd_rn (never fused
// with a neighbouring product).
H3B_DEV float2 add2_rn(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
// Two round-to-nearest products, bit-identical to two __fmul_rn.
H3B_DEV float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}

// Three-input max (sm_100): halves the instruction count of row maxima.
H3B_DEV float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Zeroes the left-out rows (bit r & 31 of keep[r >> 5] clear) of a 128-row tile
// of 128-byte rows, HALVES such tiles 16 KB apart; one warp, lane = row of 32.
// A row's 16-byte pieces keep their row under the swizzle; the lanes start at
// different pieces, so their stores meet different banks.
template <int HALVES>
H3B_DEV void zero_left_out(uint32_t tile, const uint32_t (&keep)[4], int lane) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (((keep[c] >> lane) & 1u) == 0) {
      const uint32_t row = tile + static_cast<uint32_t>(c * 32 + lane) * 128;
#pragma unroll
      for (int h = 0; h < HALVES; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(row + h * 16384 + ((i + lane) & 7) * 16), "r"(0u) : "memory");
    }
  }
}

H3B_DEV float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
H3B_DEV float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
