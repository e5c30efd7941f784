// What the products' kernels on the tensor cores share: clusters, bounded waits,
// TMA loads and MMAs of one CTA or a pair, operand descriptors.
#pragma once

#include "common.cuh"
#include "tc_ptx.cuh"

namespace es {

constexpr uint64_t kTcWaitNs = 2000000000ull;
constexpr uint64_t kTcDrainNs = 100000000ull;

enum { kKindF16 = 0, kKindI8 = 1 };

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Address of this CTA's shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t at_rank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}

__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Arrives where this thread publishes no memory (TMEM handed back, its loads done): a
// release of the whole cluster's scope would wait for the thread's global stores and
// loads, which cost the scaled 8-bit product 2000 cycles a block.
__device__ __forceinline__ void arrive_done_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ bool try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// Eight columns of this warp's TMEM lanes.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ float load_at(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// The same within the CTA's scope: for what TMA or the tensor cores signal, and TMEM
// handed back (no memory of another CTA is read behind it).
__device__ __forceinline__ bool try_wait_cta(uint64_t* bar, uint32_t parity) { return mbar_try_wait(bar, parity); }

// Bounded wait; false when this CTA has given up. Ctl: a struct in shared memory
// with `abort`, set when a wait runs out, and `progress`, a counter whose movement
// shows (where `progress` asks for it) that the wait is long and not stuck.
template <bool CTA = false, typename Ctl>
__device__ bool tc_wait(uint64_t* bar, uint32_t parity, Ctl* ctl, int32_t* status, bool progress = false) {
  auto try_wait = [&] { return CTA ? try_wait_cta(bar, parity) : try_wait_cluster(bar, parity); };
  // Within the CTA most waits are short: the timer's own latency stays out of them. Looks of
  // the cluster's scope cost more (8 bits, 16400 rows of 64 experts: 88 us with one, 92 with 64).
  for (int i = 0; i < (CTA ? 64 : 1); ++i)
    if (try_wait()) return true;
  uint64_t t0 = global_ns();
  uint32_t seen = *reinterpret_cast<volatile uint32_t*>(&ctl->progress);
  for (uint32_t i = 1;; ++i) {
    if (try_wait()) return true;
    if ((i & 31) == 0) {
      if (*reinterpret_cast<volatile int*>(&ctl->abort)) return false;
      const uint64_t now = global_ns();
      const uint32_t cur = *reinterpret_cast<volatile uint32_t*>(&ctl->progress);
      if (progress && cur != seen) {
        seen = cur;
        t0 = now;
      }
      if (now - t0 > kTcWaitNs) break;
    }
  }
  *reinterpret_cast<volatile int*>(&ctl->abort) = 1;
  if (status) *reinterpret_cast<volatile int32_t*>(status) = ES_ERR_TIMEOUT;
  return false;
}

// The wait of a whole warp: one look by all, then lane 0 waits for them.
template <bool CTA = false, typename Ctl>
__device__ __forceinline__ bool tc_wait_warp(uint64_t* bar, uint32_t parity, Ctl* ctl, int32_t* status,
                                             bool progress = false) {
  if (__all_sync(0xffffffffu, CTA ? try_wait_cta(bar, parity) : try_wait_cluster(bar, parity))) return true;
  int go = 0;
  if ((threadIdx.x & 31) == 0) go = tc_wait<CTA>(bar, parity, ctl, status, progress) ? 1 : 0;
  return __shfl_sync(0xffffffffu, go, 0) != 0;
}

__device__ inline void tc_drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = global_ns();
  for (uint32_t i = 0;; ++i) {
    if (try_wait_cluster(bar, parity)) return;
    if ((i & 31) == 0 && global_ns() - t0 > kTcDrainNs) return;
  }
}

// TMA loads; bar is a shared::cluster address (the leader's barrier, for a
// pair of CTAs), which needs the cta_group::2 form.
template <int CG>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// Four rows of a tensor into four consecutive 128-byte rows.
template <int CG>
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, int x, const int (&r)[4],
                                          uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(bar)
        : "memory");
}

// One MMA, issued by an elected lane of a converged warp.
template <int CG, int KIND>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
#define ES_MMA(group, kind)                                                                               \
  asm volatile("{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"        \
               "@e tcgen05.mma.cta_group::" #group ".kind::" #kind " [%0], %1, %2, %3, p;\n\t}" ::"r"(d), \
               "l"(a), "l"(b), "r"(idesc), "r"(accum)                                                     \
               : "memory")
  if constexpr (CG == 2 && KIND == kKindF16) ES_MMA(2, f16);
  if constexpr (CG == 2 && KIND == kKindI8) ES_MMA(2, i8);
  if constexpr (CG == 1 && KIND == kKindF16) ES_MMA(1, f16);
  if constexpr (CG == 1 && KIND == kKindI8) ES_MMA(1, i8);
#undef ES_MMA
}

// Arrives on the barrier (of both CTAs of a pair) when the MMAs that the
// elected lane has issued so far are done; a converged warp.
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::
            "r"(smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    umma_commit_warp(bar);
}

template <int CG>
__device__ __forceinline__ void tc_alloc(uint32_t* slot, uint32_t ncols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(slot, ncols);
  }
}

template <int CG>
__device__ __forceinline__ void tc_dealloc(uint32_t taddr, uint32_t ncols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
  else
    tmem_dealloc(taddr, ncols);
}

// Descriptor of an operand in 128-byte swizzled rows. K-major: rows of depth,
// 8-row groups 1024 bytes apart. MN-major: rows of 64 lanes, one row for each
// k; 8-k groups 1024 bytes apart, the next 64 lanes one box (64 k) on.
__device__ __forceinline__ uint64_t operand(uint32_t saddr, bool mn) {
  uint64_t d = static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(mn ? 8192 >> 4 : 1) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

}  // namespace es
