// fufft_tc.cuh -- tensor-core building blocks for sm_100a (inline PTX):
// tensor memory, block-scaled 4-bit products, their shared-memory and
// instruction descriptors, and TMA tiles of 128-byte rows.
#pragma once
#include "fufft_device.cuh"

namespace fufft {
namespace tc {

// ---- tensor memory ---------------------------------------------------------
// COLS: a power of two, 32 .. 512; one whole warp allocates and frees
template<int COLS> __device__ __forceinline__ void tmem_alloc(uint32_t* at_smem)
{
   asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(at_smem)), "n"(COLS) : "memory");
   asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template<int COLS> __device__ __forceinline__ void tmem_free(uint32_t at)
{
   asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(at), "n"(COLS));
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_load_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 16 consecutive columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_load16(uint32_t at, float* v)
{
   uint32_t r[16];
   asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                  "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                : "r"(at));
#pragma unroll
   for(int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// ---- descriptors -----------------------------------------------------------
// rows of 128 bytes, the 16-byte chunks of a row permuted by TMA's 128-byte
// swizzle, groups of eight rows 1024 bytes apart; `at` may step by 32 bytes
// (64 4-bit values) inside the row
__device__ __forceinline__ uint64_t rows_desc(uint32_t at)
{
   return (uint64_t)((at & 0x3ffff) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// 32 rows of 16 bytes, plain: what a 32x128b copy to tensor memory reads
__device__ __forceinline__ uint64_t scales_desc(uint32_t at)
{
   return (uint64_t)((at & 0x3ffff) >> 4) | (8ull << 32) | (1ull << 46);
}
// kind::mxf4: both operands E2M1, scales E8M0, M x N outputs; `sf` = byte (0
// or 2) of the 32-bit scale column that holds the two blocks of this step
__host__ __device__ constexpr uint32_t mxf4_idesc(int m, int n, int sf)
{
   return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27) |
          ((uint32_t)sf << 29) | ((uint32_t)sf << 4);
}

// one 512-byte scale tile (128 rows x 4 blocks) -> four columns of tensor
// memory, the same in all four 32-lane quarters
__device__ __forceinline__ void copy_scales(uint32_t to_tmem, uint64_t desc)
{
   asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" :: "r"(to_tmem), "l"(desc) : "memory");
}
// D[128 x N] (+)= A[128 x 64] B[N x 64]^T under their scales
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         bool add)
{
   asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)add) : "memory");
}
// the barrier completes when all the tensor work issued so far by this thread has
__device__ __forceinline__ void commit(uint64_t* bar)
{
   asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}

// ---- the same for a pair of CTAs (cta_group::2): one thread of the even CTA
// issues for both; A and D rows 0 .. 127 / 128 .. 255 and the halves of B's
// rows lie in the two CTAs' memories at the same addresses -----------------
template<int COLS> __device__ __forceinline__ void tmem_alloc_pair(uint32_t* at_smem)
{
   asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(at_smem)), "n"(COLS) : "memory");
   asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
template<int COLS> __device__ __forceinline__ void tmem_free_pair(uint32_t at)
{
   asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(at), "n"(COLS));
}
__device__ __forceinline__ void copy_scales_pair(uint32_t to_tmem, uint64_t desc)
{
   asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" :: "r"(to_tmem), "l"(desc) : "memory");
}
__device__ __forceinline__ void mma_mxf4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                              bool add)
{
   asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)add) : "memory");
}
// completes the barrier at this address in both CTAs
__device__ __forceinline__ void commit_pair(uint64_t* bar)
{
   asm volatile("{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
                "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
                :: "r"(smem_u32(bar)) : "memory");
}
// 2-D tile of this GPU's own memory into this CTA's shared memory, counted on
// a barrier (cluster address) of either CTA of the pair.  x: a multiple of 16 bytes
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* tm, int x, int y, uint32_t bar)
{
   asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                :: "r"(smem_u32(dst)), "l"(tm), "r"(x), "r"(y), "r"(bar) : "memory");
}

// Tensor instructions take their operands from uniform registers, and the
// thread that issues them is what a short step waits for: the whole warp runs
// the issuing loop on values that the compiler sees to be uniform
// (uniform_warp), and one lane, picked by the hardware, issues.
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0); }
__device__ __forceinline__ bool elect()
{
   uint32_t p;
   asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
   return p != 0;
}

__device__ __forceinline__ void arrive_own(uint64_t* bar)
{
   asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(smem_u32(bar)) : "memory");
}

// ---- tiles on their way out ---------------------------------------------------
// 2-D tile from shared memory; what lies outside the tensor is left out.  x, y not negative, x a multiple of 16 bytes
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* tm, int x, int y, const void* src)
{
   asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
                :: "l"(tm), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
   asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// this thread's stores have been read out of shared memory / have been done
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---- programmatic dependent launch -----------------------------------------
// the next kernel of the stream, if it was launched so, may be scheduled from here on
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }
// everything that the kernel before wrote is there (at once, if this one was launched plainly)
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- clusters --------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank()
{
   uint32_t r;
   asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
   return r;
}
// all threads of all CTAs of the cluster; orders their shared-memory accesses
__device__ __forceinline__ void cluster_sync()
{
   asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address in CTA `rank`'s shared memory of what `p` is in this one's
__device__ __forceinline__ uint32_t peer_smem(const void* p, uint32_t rank)
{
   uint32_t r;
   asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
   return r;
}
// hands no written memory over (a release of cluster scope waits for the
// thread's stores to be seen everywhere, 1100 to 1900 clocks beside tensor
// copies): for tensor memory that tcgen05.wait::ld has seen read
__device__ __forceinline__ void arrive_peer(uint32_t bar)
{
   asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" :: "r"(bar) : "memory");
}
// (volatile, but no memory clobber: several may be under way)
__device__ __forceinline__ float load_peer(uint32_t at)
{
   float v;
   asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at));
   return v;
}
__device__ __forceinline__ float4 load_peer4(uint32_t at)
{
   float4 v;
   asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
   return v;
}

}  // namespace tc
}  // namespace fufft
