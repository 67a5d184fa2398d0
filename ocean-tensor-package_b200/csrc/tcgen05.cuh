// The few instructions of the fifth-generation tensor cores that block_gemm issues, and its bounded waits.
#pragma once
#include <cstdint>
#include <cuda.h>

namespace sd { namespace tc {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count)
{
   asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar)
{
   asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes)
{
   asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
   uint32_t ok;
   asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
                : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
   return ok != 0;
}
// Every wait ends: after about two seconds (in clock cycles) it gives up and returns false.
constexpr long long WAIT_CYCLES = 4000000000ll;
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity)
{
   if (bar_try(bar, parity)) return true;
   const long long from = clock64();
   while (!bar_try(bar, parity))
      if (clock64() - from > WAIT_CYCLES) return false;
   return true;
}
// For a warp that waits as one
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, bar_wait(bar, parity)); }
// One lane of a whole warp.  The loops that issue copies and products are run by all lanes, so that addresses and
// descriptors stay in uniform registers, and only the instructions themselves by one.
__device__ __forceinline__ bool elect()
{
   uint32_t yes;
   asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xFFFFFFFF;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
   return yes != 0;
}
// The address of the same place in block `rank` of the cluster
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank)
{
   uint32_t there;
   asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
   return there;
}
// An arrival at another block's barrier.  It orders tensor memory (with tcgen05.fence around it), not shared or global
// memory, so it goes without a release for the cluster, which costs about 1000 cycles.
__device__ __forceinline__ void bar_arrive_at(uint32_t cluster_addr)
{
   asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}

// PAIR: two blocks of a cluster work on one tile of twice the rows; block 0 issues the products for both.

// A box of a two-dimensional tensor to this block's shared memory; in a pair the barrier may be block 0's
template <bool PAIR> __device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y)
{
   if (PAIR)
      asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                   :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
   else
      asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                   :: "r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}

// Rows of 128 bytes, side by side in groups of eight (1024 bytes), 128-byte swizzle, contiguous along the depth
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t addr)
{
   return (uint64_t)((addr & 0x3FFFF) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// D (+)= A B, 8-bit floating-point operands from shared memory, 32-bit sums in tensor memory, depth 32
template <bool PAIR> __device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
   if (PAIR)
      asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                   "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                   :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
   else
      asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                   "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}"
                   :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add) : "memory");
}
// Arrives on the barrier (of both blocks of a pair) when the products issued so far are done
template <bool PAIR> __device__ __forceinline__ void commit(uint32_t bar)
{
   if (PAIR)
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                   :: "r"(bar), "h"((uint16_t)3) : "memory");
   else
      asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after()  { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <bool PAIR> __device__ __forceinline__ void alloc(uint32_t where, uint32_t columns)
{
   if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(where), "r"(columns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
   } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(where), "r"(columns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
   }
}
template <bool PAIR> __device__ __forceinline__ void dealloc(uint32_t addr, uint32_t columns)
{
   if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
   else      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(addr), "r"(columns));
}

// 8, 16 or 32 columns of a warp's 32 lanes; the values may be used after ld_wait on the same registers
__device__ __forceinline__ void ld(uint32_t addr, uint32_t (&v)[8])
{
   asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                : "r"(addr));
}
__device__ __forceinline__ void ld_wait(uint32_t (&v)[8])
{
   asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]));
}
__device__ __forceinline__ void ld(uint32_t addr, uint32_t (&v)[16])
{
   asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                  "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                : "r"(addr));
}
__device__ __forceinline__ void ld_wait(uint32_t (&v)[16])
{
   asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]));
}
__device__ __forceinline__ void ld(uint32_t addr, uint32_t (&v)[32])
{
   asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                  "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
                  "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
                : "r"(addr));
}
__device__ __forceinline__ void ld_wait(uint32_t (&v)[32])
{
   asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31]));
}

// Two 32-bit operations in one instruction
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi)); return r; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }

// A warpgroup's registers a thread
template <int N> __device__ __forceinline__ void registers_up()   { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(N)); }
template <int N> __device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(N)); }

__device__ __forceinline__ void cluster_sync()
{
   asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ float4 peer_load(uint32_t addr, uint32_t rank)
{
   float4 v;
   asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at_rank(addr, rank)) : "memory");
   return v;
}

// Four bytes to shared memory without a register in between; `in` false: zero
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, bool in)
{
   asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory"); }

} } // namespace sd::tc
