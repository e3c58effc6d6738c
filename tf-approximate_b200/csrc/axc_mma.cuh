// Wrappers around the sm_100a instructions that the matrix kernels are made of: barriers, tiled bulk copies, the tensor memory and
// the matrix instruction with its descriptors.
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace axc {
namespace mma {

constexpr int kWaitPolls = 1 << 20;            // polls after which a wait gives up, about a second

__device__ __forceinline__ unsigned smem_address(const void *p) { return unsigned(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ unsigned cluster_rank()
{
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address in the cluster's window of what lies at `addr` in the CTA `rank`
__device__ __forceinline__ unsigned in_cta(unsigned addr, unsigned rank)
{
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

// true in one thread of the warp, the same one every time
__device__ __forceinline__ bool elect()
{
    unsigned yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}

__device__ __forceinline__ void barrier_init(unsigned bar, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(unsigned bar, unsigned bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// one arrival at a barrier of any CTA of the cluster (`bar` from in_cta)
__device__ __forceinline__ void barrier_arrive_cluster(unsigned bar)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The whole warp waits for the phase `parity`; false, in all its threads, when it did not come within `polls`.
__device__ __forceinline__ bool barrier_wait(unsigned bar, unsigned parity, int polls)
{
    for (int it = 0; it < polls; ++it) {
        unsigned done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (__all_sync(0xffffffffu, done != 0)) return true;
    }
    return false;
}

// One box of a tensor map, counted in bytes on `bar`.  CG 2: `bar` may lie in the other CTA of the pair.
template <int CG>
__device__ __forceinline__ void load_box(unsigned dst, const CUtensorMap *map, unsigned bar, int x, int y, int z)
{
    if constexpr (CG == 2)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                     ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map)
{
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_alloc(unsigned dst, unsigned columns)
{
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(unsigned at, unsigned columns)
{
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(at), "r"(columns));
}

// D (+)= A B^T for one K of 16, operands in shared memory, D in tensor memory
template <int CG>
__device__ __forceinline__ void multiply(unsigned d, uint64_t a, uint64_t b, unsigned shape, bool add)
{
    if constexpr (CG == 2)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(unsigned(add)) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(shape), "r"(unsigned(add)) : "memory");
}
// An arrival at `bar` (CG 2: at the same place in both CTAs) once all matrix instructions issued so far are done
template <int CG>
__device__ __forceinline__ void commit(unsigned bar)
{
    if constexpr (CG == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((unsigned short)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: x[i] = column i of this thread's row.  The values are there after load_wait().
__device__ __forceinline__ void load_columns(unsigned at, unsigned (&x)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]),
                   "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]),
                   "=r"(x[19]), "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]),
                   "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
                 : "r"(at));
}
__device__ __forceinline__ void load_columns(unsigned at, unsigned (&x)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]),
                   "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
                 : "r"(at));
}
// (the values are named, so that nothing is computed from them before)
__device__ __forceinline__ void load_wait(unsigned (&x)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]),
                   "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15]), "+r"(x[16]), "+r"(x[17]), "+r"(x[18]), "+r"(x[19]),
                   "+r"(x[20]), "+r"(x[21]), "+r"(x[22]), "+r"(x[23]), "+r"(x[24]), "+r"(x[25]), "+r"(x[26]), "+r"(x[27]), "+r"(x[28]), "+r"(x[29]),
                   "+r"(x[30]), "+r"(x[31])
                 :: "memory");
}
__device__ __forceinline__ void load_wait(unsigned (&x)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(x[0]), "+r"(x[1]), "+r"(x[2]), "+r"(x[3]), "+r"(x[4]), "+r"(x[5]), "+r"(x[6]), "+r"(x[7]), "+r"(x[8]), "+r"(x[9]),
                   "+r"(x[10]), "+r"(x[11]), "+r"(x[12]), "+r"(x[13]), "+r"(x[14]), "+r"(x[15])
                 :: "memory");
}

// the same for 64 columns
__device__ __forceinline__ void load_columns(unsigned at, unsigned (&x)[64])
{
    load_columns(at, reinterpret_cast<unsigned(&)[32]>(x[0]));
    load_columns(at + 32, reinterpret_cast<unsigned(&)[32]>(x[32]));
}
__device__ __forceinline__ void load_wait(unsigned (&x)[64])
{
    load_wait(reinterpret_cast<unsigned(&)[32]>(x[0]));
    load_wait(reinterpret_cast<unsigned(&)[32]>(x[32]));
}

// Descriptor of an operand in shared memory, 128-byte swizzle.  K contiguous: rows of 64 values, 8 rows make a group of 1024 bytes
// (stride 1024 from group to group).  Rows contiguous: 64 of them side by side, one line for each k; groups of 8 k are 1024 bytes
// apart, the next 64 rows `chunk` bytes on.  `unit`: the address in units of 16 bytes.
__device__ __forceinline__ uint64_t operand(unsigned unit, unsigned chunk)
{
    return uint64_t(unit & 0x3fffu) | (uint64_t(chunk >> 4) << 16) | (uint64_t(1024u >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// Shape of the instruction: fp32 sums of bf16 or fp16 products, M x N, operands with K or with rows contiguous
__host__ __device__ inline unsigned instruction_shape(int m, int n, bool bf16, bool a_rows, bool b_rows)
{
    return (1u << 4) | (unsigned(bf16) << 7) | (unsigned(bf16) << 10) | (unsigned(a_rows) << 15) | (unsigned(b_rows) << 16) |
           (unsigned(n >> 3) << 17) | (unsigned(m >> 4) << 24);
}

}  // namespace mma
}  // namespace axc
