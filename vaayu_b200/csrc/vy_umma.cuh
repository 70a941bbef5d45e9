// vy_umma.cuh -- barrier, TMA and tcgen05 helpers shared by the tensor-core kernels (sm_100a).
#pragma once

#include <cuda.h>

#include <mutex>

#include "vy_common.cuh"

namespace vy {

constexpr uint64_t kWaitNs = 2000000000ull;   // a barrier wait gives up after 2 s

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ── mbarrier / TMA / tcgen05 wrappers ───────────────────────────────────────────────────────

__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// The same test, but a thread whose phase is not complete yet may be suspended (woken when it
// completes) for up to `hint_ns` instead of returning at once: waiting warps then take no issue
// slots from the working ones.
__device__ __forceinline__ bool mbar_try_sleep(uint64_t* bar, uint32_t parity, uint32_t hint_ns) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(hint_ns)
        : "memory");
    return ok != 0;
}
constexpr uint32_t kSuspendNs = 100000;   // a waiting thread rechecks abort / timeout every 0.1 ms
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// Bounded wait (try_wait suspends in hardware between polls); false once the CTA has aborted, or
// after `limit_ns`, when it aborts the CTA itself (error bit 4).
__device__ __forceinline__ bool mbar_wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                              int32_t* err, uint64_t limit_ns) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = now_ns();
    for (;;) {
        if (mbar_try_sleep(bar, parity, kSuspendNs)) return true;
        if (*abort_flag) return false;
        if (now_ns() - t0 > limit_ns) {
            *abort_flag = 1;
            if (err) atomicOr(err, 4);
            return false;
        }
    }
}

__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          int32_t* err) {
    return mbar_wait_for(bar, parity, abort_flag, err, kWaitNs);
}

// Bounded wait that ignores the abort flag: drains work already issued (TMA loads, MMAs) before
// the CTA releases its shared memory and TMEM (error bit 8 if even that times out).
__device__ __forceinline__ bool mbar_drain(uint64_t* bar, uint32_t parity, int32_t* err) {
    const uint64_t t0 = now_ns();
    for (;;) {
        if (mbar_try_sleep(bar, parity, kSuspendNs)) return true;
        if (now_ns() - t0 > kWaitNs) {
            if (err) atomicOr(err, 8);
            return false;
        }
    }
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// True in one lane of a converged warp.  The loops that feed the tensor core run in whole warps and only
// the issue itself in the elected lane: around code of one lane the compiler cannot keep descriptors
// and coordinates in uniform registers, which TMA and MMA instructions take them from.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}
// A whole warp's bounded wait.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int32_t* err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err));
}

// Asks for a tile in L2.  L2 is where the writes of a kernel still running arrive too, so this is safe
// before the wait on the kernel in front, whatever that one writes.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(x), "r"(y) : "memory");
}

// A 2D tile from shared memory (what lies outside the matrix is not written), the calling thread's
// bulk group, and its waits: until shared memory has been read, or until all is written.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, int x, int y, const void* src) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y),
                 "r"(smem_u32(src))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ── tcgen05 on a CTA pair ───────────────────────────────────────────────────────────────────

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Every thread of every CTA of the cluster; shared-memory writes before it are visible after it.
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The shared::cluster address of `addr` (an address in this CTA's shared memory) in CTA `rank`.
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// A 2D tile into this CTA's shared memory whose bytes complete on a barrier of either CTA of the
// pair (`bar` is a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
        "[%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

template <int PAIR>
__device__ __forceinline__ void tmem_alloc_n(uint32_t* dst, uint32_t ncols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int PAIR>
__device__ __forceinline__ void tmem_free_n(uint32_t taddr, uint32_t ncols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
    } else {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
    }
}

// One MMA of K = 32 bytes: 16-bit floats into fp32 (I8 = false) or int8 into int32 (I8 = true),
// on one CTA or (PAIR) on the pair, issued by its first CTA.
template <bool I8, int PAIR>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
#define VY_MMA_SS(GROUP, KINDNAME)                                                                                \
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma." GROUP ".kind::" KINDNAME " [%0], %1, %2, %3, p; }" \
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)                                                   \
                 : "memory")
    if constexpr (PAIR && I8) VY_MMA_SS("cta_group::2", "i8");
    else if constexpr (PAIR) VY_MMA_SS("cta_group::2", "f16");
    else if constexpr (I8) VY_MMA_SS("cta_group::1", "i8");
    else VY_MMA_SS("cta_group::1", "f16");
#undef VY_MMA_SS
}
// Arrives on `bar` (of both CTAs of the pair whose first has cluster rank `leader`, the same offset in
// each) once every MMA this thread issued before it has completed.
__device__ __forceinline__ void mma_commit_pair(uint64_t* bar, uint32_t leader) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3u << leader))
        : "memory");
}
__device__ __forceinline__ void mma_commit_one(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle, version 1: `lbo` / `sbo` in bytes.  K-major
// tiles: rows 128 bytes apart, 8-row groups `sbo` apart (lbo unused).  MN-major tiles: blocks of
// 64 16-bit elements `lbo` apart along M/N, groups of 8 k `sbo` apart.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t(addr >> 4) & 0x3FFFull) | (uint64_t((lbo >> 4) & 0x3FFF) << 16) |
           (uint64_t((sbo >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor of mma_ss: fp32 accumulate of bf16 / fp16, or int32 accumulate of int8.
__host__ __device__ constexpr uint32_t umma_idesc(bool i8, bool bf16, uint32_t a_mn, uint32_t b_mn, uint32_t m,
                                                  uint32_t n) {
    const uint32_t c = i8 ? 2u : 1u, ab = (i8 || bf16) ? 1u : 0u;
    return (c << 4) | (ab << 7) | (ab << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// 16 / 32 consecutive fp32 (or int32) columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// Waits for this thread's TMEM loads; names the registers so that nothing reads them earlier.
__device__ __forceinline__ void tmem_wait16(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// ── host: tensor maps ───────────────────────────────────────────────────────────────────────

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn(int* status) {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    *status = fn ? VY_OK : fail(VY_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    return fn;
}

// A row-major [rows, cols] matrix (rows `ld` elements apart) of 16-bit floats or int8 as tiles of
// box_cols x box_rows with the 128-byte swizzle; what lies outside reads as zero.
inline int make_map_2d(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t cols, int64_t ld,
                       int box_cols, int box_rows) {
    int st;
    EncodeTiledFn fn = encode_tiled_fn(&st);
    if (!fn) return st;
    const CUtensorMapDataType type = dtype == VY_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : dtype == VY_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const int64_t size = dtype == VY_BF16 || dtype == VY_F16 ? 2 : 1;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld * size)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
    const cuuint32_t estr[2] = {1, 1};
    auto encode = [&] {
        return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {
        // a host thread that has made no runtime call yet (autograd's, say) has no context bound:
        // setting its current device again binds the device's primary context
        const int dev = current_device();
        if (dev < 0) return VY_ERR_CUDA;
        if (cudaSetDevice(dev) == cudaSuccess) r = encode();
    }
    if (r != CUDA_SUCCESS)
        return fail(VY_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for [%lld, %lld], row stride %lld",
                    static_cast<int>(r), (long long)rows, (long long)cols, (long long)ld);
    return VY_OK;
}

}  // namespace vy
