// Products of a feed-forward layer with many tokens, on CTA pairs (included by feed_forward.cu).
//
// Same pieces as gemm_tiles_kernel -- TMA ring, M = 256 instructions of a pair, two accumulators, K over the pairs of a cluster
// -- in three forms that clpk_gemm does not have:
//
//  * kScaled: sums of 8-bit integers with scales for each token and channel and a bias in the epilogue.
//  * kGated: two products that share A in one pass.  In a pair's instruction each CTA brings half of the tile's columns of B, so
//    the leader loads Wg's rows and its peer Wu's: columns [0, tn / 2) of the accumulator are g and [tn / 2, tn) are u of the same
//    features, a thread of the epilogue holds both, and h = act(g) * u leaves without g or u having been anywhere.
//  * kGradients: the products of the backward pass (clpk_linear_grad.cuh).
//
// What bounds it.  Long sums: the tensor cores and the card's power limit.  Gated bf16 4096^3 keeps the tensor pipe busy for 94.5 % of
// the SMs' active cycles, at 1.51 GHz; 8192 x 4096 x 8192 takes 782 to 817 us in a running program (1.34 to 1.41 PFLOPS), the
// library's plain product of that size 800 to 813 in the same minutes, and int8 8192^3 with scales and bias 389 to 393 (2.8
// POPS) where clpk_gemm's with 32-bit results takes 400.  A K block of a 256 x 256 tile is 512 tensor cycles: 0.28 us while half of
// the SMs work, 0.39 to 0.44 when all do.  Tiles of 512 rows, which fetch a quarter less, were 5 to 11 % slower in every form:
// tensor memory then holds one accumulator, and an epilogue with activations is too long to stand exposed.  Short sums: the
// epilogue, 1 us a unit of 32 x 32 results and warp (gated: two special-function results an element).
#pragma once

enum LinearForm { kGated = 0, kScaled = 1, kGradients = 2 };

constexpr int kLinearMaxStages = 12;
constexpr uint32_t kLinearM = 256;
constexpr uint32_t kLinearK = 64;                                   // of 16-bit elements: 128 bytes; 128 of the 8-bit ones
constexpr uint32_t kLinearChunk = 32;                               // columns per tcgen05.ld and per box of C
constexpr int kLinearThreads = 64 + 32 * kEpilogueWarps;

struct LinearSmem {
    uint64_t full[kLinearMaxStages];
    uint64_t empty[kLinearMaxStages];
    uint64_t tmem_full[2];
    uint64_t tmem_empty[2];
    uint32_t tmem_base;
};

// a result: h, g, u or c; dx, dWg, dWu
struct LinearResult {
    void *base;
    uint64_t ld;
    uint32_t m, n;
    uint32_t ragged;                                // its rows end inside 16 bytes
    int type;                                       // CLPK_DT_*
};

struct LinearParams {
    uint32_t tiles_m, tiles_n, group;
    uint32_t k_blocks;                              // of 128 bytes
    uint32_t tn, splits, stages, kps, tmem_cols;    // kps: K blocks per stage
    int activation;                                 // CLPK_ACT_*
    uint32_t keep;                                  // kGated: g and u are stored too
    LinearResult c[3];
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
    uint32_t *status;
};

// bytes of one K block in a CTA: its 128 rows of A and its half of the tile's columns of B
__host__ __device__ constexpr uint32_t linear_block_bytes(uint32_t tn) { return kHalfTileBytes + tn / 2 * kRowBytesK; }

__device__ __forceinline__ uint32_t pack16(float a, float b, int type)
{
    if (type == CLPK_DT_F16) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// 32 columns of one row per lane -> the warp's staging box (rows of 64 or 128 bytes in the swizzle of that width) -> one TMA
// store, which clips what lies beyond C -- in units of 16 bytes: where a row of C ends inside one, the box that holds its end is
// written element by element, so that what lies behind the row stays as it is.
__device__ __forceinline__ void linear_store(const float (&v)[32], const LinearResult &c, uint8_t *boxes, uint32_t &n_stored, const CUtensorMap *map, uint32_t col,
                                             uint32_t row, int lane)
{
    const bool wide = c.type == CLPK_DT_F32;
    // 16 bits: two 2 KiB boxes in turn: the one filled now was handed to TMA two stores ago
    uint8_t *box = wide ? boxes : boxes + (n_stored & 1) * 2048;
    if (lane == 0) {
        if (wide)
            bulk_wait_read<0>();
        else
            bulk_wait_read<1>();
    }
    __syncwarp();
    if (wide) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j++)
            *reinterpret_cast<float4 *>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const float *x = v + 8 * j;
            *reinterpret_cast<uint4 *>(box + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(pack16(x[0], x[1], c.type), pack16(x[2], x[3], c.type), pack16(x[4], x[5], c.type), pack16(x[6], x[7], c.type));
        }
    }
    if (c.ragged && col < c.n && c.n - col < kLinearChunk) {
        __syncwarp();
        const uint32_t left = c.n - col, j = lane * (wide ? 4 : 2), piece = j >> 4, in_piece = j & 15;
        const uint32_t rows = c.m > row ? (c.m - row < 32 ? c.m - row : 32) : 0;
#pragma unroll 8
        for (uint32_t i = 0; i < rows; i++) {
            const uint64_t at = (uint64_t)(row + i) * c.ld + col + lane;
            if (lane < left) {
                if (wide)
                    static_cast<float *>(c.base)[at] = *reinterpret_cast<const float *>(box + i * 128 + ((piece ^ (i & 7)) << 4) + in_piece);
                else
                    static_cast<uint16_t *>(c.base)[at] = *reinterpret_cast<const uint16_t *>(box + i * 64 + ((piece ^ ((i >> 1) & 3)) << 4) + in_piece);
            }
        }
        __syncwarp();
        if (lane == 0)
            bulk_commit();                              // an empty group: the boxes' turns are counted in groups
    } else {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(map, box, (int32_t)col, (int32_t)row);
            bulk_commit();
        }
    }
    n_stored++;
}

template <int ACT>
__device__ __forceinline__ void gate32(float (&h)[32], const float (&u)[32])
{
#pragma unroll
    for (int i = 0; i < 32; i++)
        h[i] = activate<ACT>(h[i]) * u[i];
}

__device__ __forceinline__ void gate32_by(int act, float (&h)[32], const float (&u)[32])
{
    switch (act) {
    case CLPK_ACT_SILU:      gate32<CLPK_ACT_SILU>(h, u); break;
    case CLPK_ACT_GELU_TANH: gate32<CLPK_ACT_GELU_TANH>(h, u); break;
    case CLPK_ACT_GELU:      gate32<CLPK_ACT_GELU>(h, u); break;
    case CLPK_ACT_RELU:      gate32<CLPK_ACT_RELU>(h, u); break;
    default:                 gate32<CLPK_ACT_SIGMOID>(h, u); break;
    }
}

// the sums of a chunk in fp32; those of 8-bit integers with their scales, of which lane i has that of column i
template <int DT>
__device__ __forceinline__ void scaled32(float (&v)[32], const uint32_t (&sum)[32], float row_scale, float col_scale)
{
#pragma unroll
    for (int i = 0; i < 32; i++) {
        if constexpr (DT == CLPK_DT_I8)
            v[i] = (float)(int32_t)sum[i] * row_scale * __shfl_sync(0xffffffffu, col_scale, i);
        else
            v[i] = __uint_as_float(sum[i]);
    }
}

__device__ __forceinline__ float bias_at(const void *bias, int type, uint32_t col)
{
    if (type == CLPK_DT_F32)
        return static_cast<const float *>(bias)[col];
    return type == CLPK_DT_F16 ? __half2float(static_cast<const __half *>(bias)[col]) : __bfloat162float(static_cast<const __nv_bfloat16 *>(bias)[col]);
}

// What a unit of 8-bit sums is finished with: the scale of the lane's row, and of column `col` + lane those of the one or two
// products, or scale and bias.  They are asked for a unit ahead.
struct LinearScales {
    float row = 1.0f, col0 = 1.0f, col1 = 0.0f;

    template <int DT, LinearForm FORM>
    __device__ __forceinline__ void rows(const LinearParams &p, uint32_t row0, int lane)
    {
        if constexpr (DT == CLPK_DT_I8)
            row = row0 + lane < p.c[0].m ? p.a_scale[row0 + lane] : 0.0f;
    }
    template <int DT, LinearForm FORM>
    __device__ __forceinline__ void cols(const LinearParams &p, uint32_t first, int lane)
    {
        if constexpr (DT == CLPK_DT_I8) {
            const uint32_t c = first + lane;
            const bool there = c < p.c[0].n;
            col0 = there ? p.b_scale[c] : 0.0f;
            if constexpr (FORM == kGated)
                col1 = there ? p.u_scale[c] : 0.0f;
            else
                col1 = p.bias && there ? bias_at(p.bias, p.c[0].type, c) : 0.0f;
        }
    }
};

// What becomes of a unit of sums: one chunk of 32 columns, or with kGated the chunk of g and that of u.  `which`: the result
// that plain sums (kGradients) belong to.
template <int DT, LinearForm FORM>
__device__ __forceinline__ void linear_finish(const CUtensorMap *maps, const LinearParams &p, const LinearScales &scales, const uint32_t (&s0)[32],
                                              const uint32_t (&s1)[32], uint32_t which, uint32_t row, uint32_t col, uint8_t *boxes, uint32_t &n_stored, int lane)
{
    float v[32];
    scaled32<DT>(v, s0, scales.row, scales.col0);
    if constexpr (FORM == kGated) {
        float u[32];
        scaled32<DT>(u, s1, scales.row, scales.col1);
        if (p.keep) {
            linear_store(v, p.c[1], boxes, n_stored, maps + 1, col, row, lane);
            linear_store(u, p.c[2], boxes, n_stored, maps + 2, col, row, lane);
        }
        gate32_by(p.activation, v, u);
    } else if constexpr (FORM == kScaled) {
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < 32; i++)
                v[i] += __shfl_sync(0xffffffffu, scales.col1, i);
        }
    }
    linear_store(v, p.c[which], boxes, n_stored, maps + which, col, row, lane);
}

// a tile: which result, where in it (rows of 256, and for the result; columns of tn), and which K blocks of it this pair adds
struct LinearTile {
    uint32_t which, mb, mb_out, nb, kb0, kb1;
};

#include "clpk_linear_grad.cuh"

struct LinearMaps {
    CUtensorMap a, b[2], c[3];
};
template <LinearForm FORM> using LinearMapsOf = std::conditional_t<FORM == kGradients, GradMaps, LinearMaps>;
template <LinearForm FORM> using LinearParamsOf = std::conditional_t<FORM == kGradients, GradParams, LinearParams>;

// the i-th tile of a cluster; false: it has no more
template <LinearForm FORM>
__device__ __forceinline__ bool linear_tile(const LinearParamsOf<FORM> &p, uint32_t cluster, uint32_t clusters, uint32_t split, uint32_t i, LinearTile &t)
{
    if constexpr (FORM == kGradients) {
        return grad_tile(p, cluster, clusters, i, t);
    } else {
        const uint32_t tile = cluster + i * clusters;
        if (tile >= p.tiles_m * p.tiles_n)
            return false;
        dense_tile_coords(tile, p.tiles_m, p.tiles_n, p.group, t.mb, t.nb);
        t.mb_out = t.mb;
        t.which = 0;
        t.kb0 = split * p.k_blocks / p.splits;
        t.kb1 = (split + 1) * p.k_blocks / p.splits;
        return true;
    }
}

template <int DT, LinearForm FORM>
__global__ void __launch_bounds__(kLinearThreads) linear_kernel(const __grid_constant__ LinearMapsOf<FORM> maps, const __grid_constant__ LinearParamsOf<FORM> p)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t block_bytes = linear_block_bytes(p.tn), stage_bytes = p.kps * block_bytes;
    uint8_t *staging = smem + (size_t)p.stages * stage_bytes;
    LinearSmem *sh = reinterpret_cast<LinearSmem *>(staging + kEpilogueWarps * kStagingBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank(), r = rank & 1, leader = rank & ~1u, split = rank >> 1;
    const uint32_t cluster = blockIdx.x / (2 * p.splits), clusters = gridDim.x / (2 * p.splits);

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; s++) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        for (int acc = 0; acc < 2; acc++) {
            mbar_init(&sh->tmem_full[acc], 1);
            mbar_init(&sh->tmem_empty[acc], 2 * kEpilogueWarps);
        }
        mbar_fence_init();
        if constexpr (FORM != kGradients) {
            tma_prefetch_desc(&maps.a);
            tma_prefetch_desc(&maps.b[FORM == kGated ? r : 0]);
            tma_prefetch_desc(&maps.c[0]);
        }
    }
    if (warp == 1)
        tmem_alloc<2>(&sh->tmem_base, p.tmem_cols);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    griddep_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *p.status = 0u;
    griddep_launch_dependents();

    const uint32_t q = (uint32_t)(warp & 3), half = (uint32_t)(warp - 2) >> 2;     // epilogue warps
    const uint32_t unit_cols = FORM == kGated ? p.tn / 2 : p.tn, units = unit_cols / kLinearChunk;
    constexpr uint32_t kSubs = FORM == kGated ? 2 : 1;                             // chunks per unit, tn / 2 columns apart
    uint8_t *boxes = staging + (size_t)(warp - 2) * kStagingBytes;
    uint32_t n_stored = 0;
    LinearTile t;

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        const uint32_t full0 = cluster_addr(&sh->full[0], leader);
        uint32_t s = 0, parity = 1;                            // parity of the empty barrier's previous phase
        bool ok = true;
        for (uint32_t i = 0; ok && linear_tile<FORM>(p, cluster, clusters, split, i, t); i++) {
            const uint32_t row_a = t.mb * kLinearM + r * 128;
            const uint32_t row_b = FORM == kGated ? t.nb * (p.tn / 2) : t.nb * p.tn + r * (p.tn / 2);
            const uint32_t kb0 = t.kb0, kb1 = t.kb1;
            for (uint32_t kb = kb0; kb < kb1; kb += p.kps) {
                const uint32_t nk = kb1 - kb < p.kps ? kb1 - kb : p.kps;
                if (!warp_wait(&sh->empty[s], parity)) {       // a fresh barrier's preceding phase counts as complete
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x301u);
                    ok = false;
                    break;
                }
                uint8_t *st = smem + (size_t)s * stage_bytes;
                if (elect_one()) {
                    if (r == 0)
                        mbar_expect_tx(&sh->full[s], nk * 2 * block_bytes);
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++)
                        if (h < nk) {
                            uint8_t *blk = st + h * block_bytes;
                            if constexpr (FORM == kGradients) {
                                grad_load(maps, p, t.which, blk, kb + h, row_a, row_b, full0 + 8 * s);
                            } else {
                                tma_load_pair_at(blk, &maps.a, (int32_t)((kb + h) * kRowBytesK), (int32_t)row_a, full0 + 8 * s);
                                tma_load_pair_at(blk + kHalfTileBytes, &maps.b[FORM == kGated ? r : 0], (int32_t)((kb + h) * kRowBytesK), (int32_t)row_b, full0 + 8 * s);
                            }
                        }
                }
                __syncwarp();
                if (++s == p.stages) {
                    s = 0;
                    parity ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (the pair's leader) ----------------
        if (r == 0) {
            constexpr uint32_t kFmt = DT == CLPK_DT_BF16 ? kFmtBF16 : DT == CLPK_DT_F16 ? kFmtF16 : kFmtS8;
            const uint16_t pair_mask = (uint16_t)(3u << leader);
            uint32_t s = 0, parity = 0;
            bool ok = true;
            for (uint32_t i = 0; ok && linear_tile<FORM>(p, cluster, clusters, split, i, t); i++) {
                const uint32_t acc = i & 1, use = i >> 1;
                const uint32_t kb0 = t.kb0, kb1 = t.kb1;
                if (use > 0 && !warp_wait(&sh->tmem_empty[acc], (use - 1) & 1)) {
                    if (lane == 0)
                        atomicCAS(p.status, 0u, 0x302u);
                    break;
                }
                tc_fence_after_sync();
                const uint32_t d = tmem + acc * p.tn;
                const bool a_mn = FORM == kGradients && t.which > 0;       // A contiguous along M
                const uint32_t idesc = make_idesc(256, p.tn, kFmt, kFmt, DT == CLPK_DT_I8 ? kAccS32 : kAccF32) | (a_mn ? kMajorA : 0u) |
                                       (FORM == kGradients ? kMajorB : 0u);
                const uint32_t a_lbo = a_mn ? kMnLead : 16, a_step = a_mn ? kMnStep : 2;
                constexpr uint32_t kBLbo = FORM == kGradients ? kMnLead : 16, kBStep = FORM == kGradients ? kMnStep : 2;
                for (uint32_t kb = kb0; kb < kb1; kb += p.kps) {
                    if (!warp_wait(&sh->full[s], parity)) {
                        if (lane == 0)
                            atomicCAS(p.status, 0u, 0x303u);
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t base = smem_u32(smem + (size_t)s * stage_bytes);
                    const uint32_t nk = kb1 - kb < p.kps ? kb1 - kb : p.kps;
                    const uint32_t s_now = s;
                    if (++s == p.stages) {
                        s = 0;
                        parity ^= 1;
                    }
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t h = 0; h < 2; h++) {
                            if (h >= nk)
                                break;
                            const uint32_t blk = base + h * block_bytes;
                            const uint64_t ad = make_smem_desc(blk, a_lbo, 1024, kSwizzle128B), bd = make_smem_desc(blk + kHalfTileBytes, kBLbo, 1024, kSwizzle128B);
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; kk++) {
                                const uint32_t accumulate = (kb != kb0 || h != 0 || kk != 0) ? 1u : 0u;
                                if constexpr (DT == CLPK_DT_I8)
                                    mma2_i8_ss(d, ad + kk * a_step, bd + kk * kBStep, idesc, accumulate);
                                else
                                    mma2_f16_ss(d, ad + kk * a_step, bd + kk * kBStep, idesc, accumulate);
                            }
                        }
                        tc_commit_pair(&sh->empty[s_now], pair_mask);
                    }
                    __syncwarp();
                }
                if (ok && elect_one())
                    tc_commit_pair(&sh->tmem_full[acc], pair_mask);
                __syncwarp();
            }
        }
    } else if (p.splits == 1) {
        // ---------------- epilogue, K not split: the two warps of a lane quarter take every other unit ----------------
        for (uint32_t i = 0; linear_tile<FORM>(p, cluster, clusters, split, i, t); i++) {
            const uint32_t acc = i & 1, use = i >> 1;
            const uint32_t row = t.mb_out * kLinearM + r * 128 + q * 32, col = t.nb * unit_cols;
            // the two chunks that a step reads are g and u of one unit (kGated), or two units
            constexpr uint32_t kStep = FORM == kGated ? 2 : 4;
            LinearScales scales[2];
            for (int o = 0; o < 2; o++) {
                scales[o].rows<DT, FORM>(p, row, lane);
                if (o == 0 || FORM != kGated)
                    scales[o].cols<DT, FORM>(p, col + (half + 2 * o) * kLinearChunk, lane);
            }
            if (!warp_wait(&sh->tmem_full[acc], use & 1)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x304u);
                break;
            }
            tc_fence_after_sync();
            const uint32_t taddr = tmem + acc * p.tn + ((q * 32) << 16);
            auto release = [&]() {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive_cluster_relaxed(&sh->tmem_empty[acc], leader);
            };
            if (half >= units) {
                release();
                continue;
            }
            for (uint32_t c = half; c < units; c += kStep) {
                const bool two = FORM != kGated && c + 2 < units;
                uint32_t s0[32], s1[32];
                tmem_ld_32x32b_x32(taddr + c * kLinearChunk, s0);
                if (FORM == kGated || two)
                    tmem_ld_32x32b_x32(taddr + (FORM == kGated ? p.tn / 2 + c * kLinearChunk : (c + 2) * kLinearChunk), s1);
                tmem_ld_wait();
                if (c + kStep >= units)
                    release();
                LinearScales next[2] = {scales[0], scales[1]};
                if (c + kStep < units)
                    for (int o = 0; o < (FORM == kGated ? 1 : 2); o++)
                        next[o].cols<DT, FORM>(p, col + (c + kStep + 2 * o) * kLinearChunk, lane);
                linear_finish<DT, FORM>(maps.c, p, scales[0], s0, s1, t.which, row, col + c * kLinearChunk, boxes, n_stored, lane);
                if (two)
                    linear_finish<DT, FORM>(maps.c, p, scales[1], s1, s1, t.which, row, col + (c + 2) * kLinearChunk, boxes, n_stored, lane);
                scales[0] = next[0];
                scales[1] = next[1];
            }
        }
    } else if (!warp_wait(&sh->tmem_full[0], 0)) {
        if (lane == 0)
            atomicCAS(p.status, 0u, 0x305u);
    }

    if (FORM != kGradients && p.splits > 1) {
        // ---------------- K split over the cluster's pairs (one tile per cluster) ----------------
        // Every pair's instructions have retired, so the stages of the ring are free to take partial sums: slot (src, j) of CTA
        // (owner, r) holds pair src's sums of the owner's j-th unit, src counted without the owner.  They are added in the order
        // of the pairs, whoever owns the unit.
        constexpr uint32_t kUnitBytes = kSubs * kLinearChunk * 128 * 4;
        tc_fence_before_sync();
        __syncwarp();
        cluster_sync();
        tc_fence_after_sync();
        const uint32_t slots = (units + p.splits - 1) / p.splits;
        const uint32_t taddr = tmem + ((q * 32) << 16), my_row = q * 32 + lane;
        const bool epilogue = warp >= 2;
        if (epilogue) {
            for (uint32_t i = half; i < kSubs * units; i += 2) {
                const uint32_t c = i / kSubs, sub = i % kSubs, owner = c % p.splits;
                if (owner == split)
                    continue;
                uint32_t v[32];
                tmem_ld_32x32b_x32(taddr + sub * (p.tn / 2) + c * kLinearChunk, v);
                tmem_ld_wait();
                const uint32_t src = split < owner ? split : split - 1;
                const uint32_t dst = cluster_addr(smem + (size_t)(src * slots + c / p.splits) * kUnitBytes + sub * (kUnitBytes / kSubs) + my_row * 16, owner * 2 + r);
#pragma unroll
                for (uint32_t g = 0; g < 8; g++)
                    st_cluster_v4(dst + g * 2048, v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
            }
        }
        __syncwarp();
        cluster_sync();
        if (epilogue && linear_tile<FORM>(p, cluster, clusters, split, 0, t)) {
            const uint32_t row = t.mb_out * kLinearM + r * 128 + q * 32;
            for (uint32_t j = half; split + j * p.splits < units; j += 2) {
                const uint32_t c = split + j * p.splits;
                LinearScales scales;
                scales.rows<DT, FORM>(p, row, lane);
                scales.cols<DT, FORM>(p, t.nb * unit_cols + c * kLinearChunk, lane);
                uint32_t sum[2][32];
#pragma unroll
                for (uint32_t sub = 0; sub < kSubs; sub++) {
                    uint32_t own[32];
                    tmem_ld_32x32b_x32(taddr + sub * (p.tn / 2) + c * kLinearChunk, own);
                    tmem_ld_wait();
                    for (uint32_t src = 0; src < p.splits; src++) {
                        const uint8_t *slot = smem + (size_t)((src < split ? src : src - 1) * slots + j) * kUnitBytes + sub * (kUnitBytes / kSubs) + my_row * 16;
#pragma unroll
                        for (uint32_t g = 0; g < 8; g++) {
                            uint4 v = make_uint4(own[4 * g], own[4 * g + 1], own[4 * g + 2], own[4 * g + 3]);
                            if (src != split)
                                v = *reinterpret_cast<const uint4 *>(slot + g * 2048);
                            const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (uint32_t l = 0; l < 4; l++) {
                                uint32_t &x = sum[sub][4 * g + l];
                                if (src == 0)
                                    x = e[l];
                                else if constexpr (DT == CLPK_DT_I8)
                                    x += e[l];
                                else
                                    x = __float_as_uint(__uint_as_float(x) + __uint_as_float(e[l]));
                            }
                        }
                    }
                }
                linear_finish<DT, FORM>(maps.c, p, scales, sum[0], sum[kSubs - 1], t.which, row, t.nb * unit_cols + c * kLinearChunk, boxes, n_stored, lane);
            }
        }
    }
    // the staging boxes must have been read before this CTA's shared memory goes away
    if (warp >= 2 && lane == 0)
        bulk_wait_read<0>();

    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    if (warp == 1)
        tmem_dealloc<2>(tmem, p.tmem_cols);
}

// ---- host side -----------------------------------------------------------------------------

// a row-major matrix, in boxes of 128 bytes of a row times box_rows rows
static int make_matrix_map(CUtensorMap *map, const void *base, uint64_t rows, uint64_t row_bytes, uint64_t pitch_bytes, uint32_t box_rows)
{
    EncodeTiledFn enc = nullptr;
    const int rc = get_encode_fn(&enc);
    if (rc != CLPK_OK)
        return rc;
    const cuuint64_t dims[2] = {row_bytes, rows}, strides[1] = {pitch_bytes};
    const cuuint32_t box[2] = {kRowBytesK, box_rows}, estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
        return CLPK_ERR_CUDA;
    }
    return CLPK_OK;
}

// a result, in boxes of 32 x 32
static int make_result_map(CUtensorMap *map, const LinearResult &c)
{
    EncodeTiledFn enc = nullptr;
    const int rc = get_encode_fn(&enc);
    if (rc != CLPK_OK)
        return rc;
    const uint32_t elem = c.type == CLPK_DT_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {c.n, c.m}, strides[1] = {c.ld * elem};
    const cuuint32_t box[2] = {kLinearChunk, 32}, estr[2] = {1, 1};
    const CUresult r = enc(map, elem == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c.base, dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, elem == 4 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled (result) failed with CUresult %d", (int)r);
        return CLPK_ERR_CUDA;
    }
    return CLPK_OK;
}
