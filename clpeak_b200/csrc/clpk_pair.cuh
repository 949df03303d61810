// What the kernels that multiply on CTA pairs (gemm.cu, feed_forward.cu) have in common: operand tiles of 128 bytes of K per row
// brought by TMA, roles that are whole warps with one elected lane, the order of the tiles, and the boxes in which results leave.
#pragma once

#include <cuda.h>

#include "clpk_internal.h"
#include "clpk_ptx.cuh"

namespace clpk {

constexpr uint32_t kRowBytesK = 128;                        // K bytes per row per stage
constexpr uint32_t kHalfTileBytes = 128 * kRowBytesK;       // 16 KiB: 128 rows x 128 B

// 2-D tile load whose completion bytes go to the pair's leader CTA: leader_bar is its barrier's address (leader_addr).
__device__ __forceinline__ void tma_load_pair_at(void *smem_dst, const CUtensorMap *tmap, int32_t x, int32_t y,
                                                 uint32_t leader_bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(leader_bar), "r"(x), "r"(y)
        : "memory");
}

// 2-D tile load into this CTA's shared memory, its bytes counted by this CTA's barrier
__device__ __forceinline__ void tma_load_own(void *smem_dst, const CUtensorMap *tmap, int32_t x, int32_t y, uint64_t *bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(smem_dst)),
        "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y)
        : "memory");
}

__device__ __forceinline__ uint32_t leader_addr(const void *p)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(smem_u32(p)));
    return a;
}

// Roles that issue TMA or tcgen05 instructions run their loops with the whole warp and let
// one elected lane issue.  Addresses and descriptors are then warp-uniform values, which is
// what those instructions take.  With the loop inside `if (lane == 0)` each instruction cost
// its thread 110-130 cycles (measured with clock64 around it: four MMAs 460 cycles, against
// 115 this way), and a thread that must issue four MMAs and a commit per 512 tensor-core
// cycles, or eight and a commit per 1024, was the slowest stage of the pipeline.
// warp_wait: every lane waits; the verdict is made uniform so that the warp stays together.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity) ? 1 : 0) != 0;
}

// Where a wait has run out, whoever consumed the stages of a ring may have given up while loads into them are on their way: they have
// to land before the CTA's shared memory goes away.  Only a stage's last use can be on its way; each wait has its limit.
__device__ __forceinline__ void ring_settled(uint64_t *full, uint32_t stages, uint32_t issued)
{
    for (uint32_t use = issued > stages ? issued - stages : 0; use < issued; use++)
        warp_wait(&full[use % stages], use / stages & 1);
}

constexpr int kEpilogueWarps = 8;
constexpr uint32_t kStagingBytes = 32 * 128;                       // 32 rows x 128 bytes of C

// Tiles are walked in groups of `group` tile columns, M fastest inside a group.
__device__ __forceinline__ void dense_tile_coords(uint32_t tile, uint32_t tiles_m, uint32_t tiles_n, uint32_t group,
                                                  uint32_t &mb, uint32_t &nb)
{
    const uint32_t per_group = group * tiles_m;
    const uint32_t g = tile / per_group;
    const uint32_t within = tile - g * per_group;
    const uint32_t first_n = g * group;
    const uint32_t width = (tiles_n - first_n) < group ? (tiles_n - first_n) : group;
    mb = within / width;
    nb = first_n + within % width;
}

// one staging box out: wait until the previous store has read the box, fill it, hand it to TMA
__device__ __forceinline__ void store_staged_box(const uint32_t (&w)[32], uint8_t *box, const CUtensorMap *tmap_c, uint32_t col,
                                                 uint32_t row, int lane)
{
    uint8_t *my_row = box + lane * 128;
    const uint32_t sw = (uint32_t)(lane & 7);
    if (lane == 0)
        bulk_wait_read<0>();
    __syncwarp();
#pragma unroll
    for (uint32_t j = 0; j < 8; j++)
        *reinterpret_cast<uint4 *>(my_row + ((j ^ sw) << 4)) = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
        tma_store_2d(tmap_c, box, (int32_t)col, (int32_t)row);
        bulk_commit();
    }
}

__device__ __forceinline__ void st_cluster_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v)
{
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

__device__ __forceinline__ uint32_t cluster_addr(const void *p, uint32_t cta)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
    return a;
}

// ---- host side -----------------------------------------------------------------------------

constexpr uint32_t kSmemMax = 227 * 1024;           // that a CTA may have

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

static inline int get_encode_fn(EncodeTiledFn *out)
{
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void *sym = nullptr;
        cudaDriverEntryPointQueryResult qres;
        CLPK_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres));
        if (qres != cudaDriverEntryPointSuccess || !sym) {
            set_error("cuTensorMapEncodeTiled is not available from this driver");
            return CLPK_ERR_CUDA;
        }
        fn = reinterpret_cast<EncodeTiledFn>(sym);
    }
    *out = fn;
    return CLPK_OK;
}

// CTAs in clusters of `cluster`, behind the kernel before them
template <typename Maps, typename Params>
static inline int launch_clusters(void (*kernel)(Maps, Params), const char *what, uint32_t ctas, int threads, size_t smem, uint32_t cluster, cudaStream_t s,
                                  const Maps &maps, const Params &p)
{
    CLPK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = tuning(CLPK_TUNE_GEMM_NO_PDL) == 1 ? 0 : 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, maps, p);
    return e == cudaSuccess ? CLPK_OK : cuda_fail(e, what);
}

} // namespace clpk
