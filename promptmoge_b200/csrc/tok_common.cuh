// Shared pieces of the token operators (16-bit floating-point matrix products and attention on tcgen05): element types,
// the kind::f16 descriptors, matrix products whose left operand lies in tensor memory, wide tensor-memory transfers,
// packed fp32 arithmetic and tensor maps of 16-bit tensors.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace pmg {
namespace tok {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
    static constexpr int kFmt = 1;               // operand format of kind::f16
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Elem<__half> {
    static constexpr int kFmt = 0;
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<__half2*>(&v));
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// Two fp32 operations in one instruction (sm_100).
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x) {
    const float2 f = unpack2(x);
    return pack2(ex2(f.x), ex2(f.y));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The larger; NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// kind::f16 instruction descriptor: D = fp32, A and B of one 16-bit format, operands K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc16(int fmt, int M, int N, bool a_mn, bool b_mn) {
    return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Shared-memory operand in the 128-byte swizzle that TMA writes (rows of 64 16-bit values).  K-major: a row is 64
// values of K of one M / N index, 8-row groups 1024 bytes apart, the next 64 of K in the next sub-tile.  MN-major: a
// row is 64 values of M / N at one K, 8-row groups (8 of K) 1024 bytes apart, the next 64 of M / N `lbo` bytes on.
// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}

// The MMAs are issued by a converged warp, predicated on one lane (`lead`): their operands then stay in uniform
// registers, and descriptors are a constant upper word and a lower word that an addition moves along the operand.
// From one lane of a diverged warp, with descriptors put together for each, an instruction took about 90 cycles to issue.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) {
    return ((addr >> 4) & 0x3FFF) | ((lbo >> 4) << 16);
}
__device__ __forceinline__ void mma16(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(lead)
        : "memory");
}
// Left operand in tensor memory: lane = row, one 32-bit column holds two consecutive values of K.
__device__ __forceinline__ void mma16_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_commit_if(uint32_t lead, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(lead)
        : "memory");
}

// A pair of CTAs on one tile (cta_group::2): each holds its rows of A, half the rows of B and its rows of the result.  The
// even CTA issues; loads of either signal its barrier, and what it commits arrives in both.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of `bar` in the even CTA.
__device__ __forceinline__ uint32_t even_bar(uint64_t* bar) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(bar)));
    return r;
}
__device__ __forceinline__ void arrive_even(uint64_t* bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(even_bar(bar)) : "memory");
}
__device__ __forceinline__ void tma_tile2d_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma16_pair(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void commit_pair_if(uint32_t lead, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(
            smem_u32(bar)),
        "r"(lead), "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// 32 columns of this thread's tensor-memory lane; no wait (tmem_wait_ld before the values are used).
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void tmem_st16(uint32_t t, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(t),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 3-D TMA tile load at (x, y, z).
__device__ __forceinline__ void tma_tile3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// Bounded wait by polling: false on timeout or when another warp already aborted.  A softmax step is a chain of such waits;
// suspending between polls, as long waits should, cost it 2 to 6 %.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = 0;
    for (uint32_t i = 1;; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63) == 0) {
            if (*abort_flag) return false;
            const uint64_t now = global_ns();
            if (t0 == 0) t0 = now;
            if (now - t0 > kWaitNs) return false;
        }
    }
}

// After an abort: waits (bounded) until every MMA this thread issued has retired, so that tensor memory may be freed, and as
// long again as copies into shared memory take many times over: the block must not leave while one may still land, in what is
// another block's by then.  Loaders stop at their next wait, a few microseconds after the abort at most; where the issuer
// came to its end instead it has waited for all that they sent.
constexpr uint64_t kLandNs = 1000000;
template <bool PAIR = false>
__device__ __forceinline__ void drain_mma(uint64_t* bar) {
    if constexpr (PAIR) commit_pair_if(1, bar);
    else mma_commit(bar);
    const uint64_t t0 = global_ns();
    while (!mbar_try_wait_sleep(bar, 0, 4000) && global_ns() - t0 < kWaitNs) {
    }
    const uint64_t t1 = global_ns();
    while (global_ns() - t1 < kLandNs) {
    }
}

}  // namespace tok

// Host: launches a kernel that follows another of the same call.  It starts with pdl_begin(), so its launch may be
// prepared while that one runs; it waits there until that one is complete.
// CLUSTER: CTAs of a cluster.
template <int CLUSTER = 1, typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, A... args) {
    cudaLaunchAttribute attr[2];
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CLUSTER;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = CLUSTER > 1 ? 2 : 1;
    PMG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
    return PMG_OK;
}

// Host: tensor map of a 16-bit tensor (rank 2 or 3; dims and box innermost first, strides in bytes of dims 1..rank-1),
// 128-byte swizzle, zero fill out of bounds; box[0] is 64.  Base and strides 16-byte aligned.  PMG_OK or an error.
int make_tensor_map16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const uint64_t* strides,
                      const uint32_t* box);

}  // namespace pmg
