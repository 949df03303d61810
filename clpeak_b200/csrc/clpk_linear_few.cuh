// Products of a feed-forward layer with few tokens (included by feed_forward.cu).
//
// Every weight is read once and multiplied by a handful of tokens, so the time is that of reading the weights.  The operands
// change places: a tile's 128 rows are rows of the weight, as they lie in memory, and the tokens are its columns (16 to 128, the
// fewest that a tcgen05 instruction of 128 rows takes), so that of the shared memory that TMA fills nearly all is weight.  With
// kGated a tile is 64 rows of Wg above the same 64 of Wu.
//
// K is split over the CTAs of a cluster, as far as it takes to give every SM some: one tile per cluster, each CTA a K range.  Then
// the partial sums go to shared memory, [token][row of the weight], and each CTA adds and finishes the tokens of its turn, reading
// the others' sums through distributed shared memory, in the order of K.  Nothing goes through global memory.
// CTAs are small (128 threads, a ring of 64 KiB): several share an SM, and one's set-up and exchange lie under another's loads.
#pragma once

constexpr int kFewThreads = 128;
constexpr int kFewMaxStages = 8;
constexpr uint32_t kFewRows = 128;

struct FewSmem {
    uint64_t full[kFewMaxStages];
    uint64_t empty[kFewMaxStages];
    uint64_t done;
    uint32_t tmem_base;
};

struct FewMaps {
    CUtensorMap w[2], x;
};

struct FewParams {
    uint32_t m, n;                                  // tokens, rows of a weight
    uint32_t k_blocks, splits, stages, tokens;      // tokens: m rounded up to what the instruction takes
    uint32_t tmem_cols;
    int out, activation;
    void *c, *g, *u;                                // g, u: kept where not NULL
    uint64_t ldc;
    const float *a_scale, *b_scale, *u_scale;
    const void *bias;
    uint32_t *status;
};

// N neighbouring results of one token
template <int N>
__device__ __forceinline__ void few_store(void *base, int type, uint64_t at, uint32_t left, const float (&v)[N])
{
    if (type == CLPK_DT_F32) {
        float *c = static_cast<float *>(base) + at;
        if (left >= N) {
            if constexpr (N == 4)
                *reinterpret_cast<float4 *>(c) = make_float4(v[0], v[1], v[2], v[3]);
            else
                *reinterpret_cast<float2 *>(c) = make_float2(v[0], v[1]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (i < left)
                    c[i] = v[i];
        }
        return;
    }
    uint16_t *c = static_cast<uint16_t *>(base) + at;
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2)
        w[i / 2] = pack16(v[i], v[i + 1], type);
    if (left >= N) {
        if constexpr (N == 4)
            *reinterpret_cast<uint2 *>(c) = make_uint2(w[0], w[1]);
        else
            *reinterpret_cast<uint32_t *>(c) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < left)
                c[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
    }
}

__device__ __forceinline__ float activate_by(int act, float g)
{
    switch (act) {
    case CLPK_ACT_SILU:      return activate<CLPK_ACT_SILU>(g);
    case CLPK_ACT_GELU_TANH: return activate<CLPK_ACT_GELU_TANH>(g);
    case CLPK_ACT_GELU:      return activate<CLPK_ACT_GELU>(g);
    case CLPK_ACT_RELU:      return activate<CLPK_ACT_RELU>(g);
    default:                 return activate<CLPK_ACT_SIGMOID>(g);
    }
}

template <int DT, LinearForm FORM>
__global__ void __launch_bounds__(kFewThreads) linear_few_kernel(const __grid_constant__ FewMaps maps, FewParams p)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t stage_bytes = kHalfTileBytes + p.tokens * kRowBytesK;
    FewSmem *sh = reinterpret_cast<FewSmem *>(smem + (size_t)p.stages * stage_bytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t split = cluster_ctarank(), tile = blockIdx.x / p.splits;
    const uint32_t kb0 = split * p.k_blocks / p.splits, kb1 = (split + 1) * p.k_blocks / p.splits;
    constexpr uint32_t kTileCols = FORM == kGated ? 64 : 128;                       // features per tile

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; s++) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        mbar_init(&sh->done, 1);
        mbar_fence_init();
        tma_prefetch_desc(&maps.w[0]);
        tma_prefetch_desc(&maps.x);
        if constexpr (FORM == kGated)
            tma_prefetch_desc(&maps.w[1]);
    }
    if (warp == 1)
        tmem_alloc<1>(&sh->tmem_base, p.tmem_cols);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    griddep_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0)
        *p.status = 0u;
    griddep_launch_dependents();

    if (warp == 0) {
        // ---------------- TMA producer ----------------
        uint32_t s = 0, parity = 1;
        for (uint32_t kb = kb0; kb < kb1; kb++) {
            if (!warp_wait(&sh->empty[s], parity)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x311u);
                break;
            }
            uint8_t *st = smem + (size_t)s * stage_bytes;
            const int32_t x = (int32_t)(kb * kRowBytesK), row = (int32_t)(tile * kTileCols);
            if (elect_one()) {
                mbar_expect_tx(&sh->full[s], stage_bytes);
                tma_load_own(st, &maps.w[0], x, row, &sh->full[s]);
                if constexpr (FORM == kGated)
                    tma_load_own(st + kHalfTileBytes / 2, &maps.w[1], x, row, &sh->full[s]);
                tma_load_own(st + kHalfTileBytes, &maps.x, x, 0, &sh->full[s]);
            }
            __syncwarp();
            if (++s == p.stages) {
                s = 0;
                parity ^= 1;
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        constexpr uint32_t kFmt = DT == CLPK_DT_BF16 ? kFmtBF16 : DT == CLPK_DT_F16 ? kFmtF16 : kFmtS8;
        const uint32_t idesc = make_idesc(128, p.tokens, kFmt, kFmt, DT == CLPK_DT_I8 ? kAccS32 : kAccF32);
        uint32_t s = 0, parity = 0;
        bool ok = true;
        for (uint32_t kb = kb0; kb < kb1; kb++) {
            if (!warp_wait(&sh->full[s], parity)) {
                if (lane == 0)
                    atomicCAS(p.status, 0u, 0x312u);
                ok = false;
                break;
            }
            tc_fence_after_sync();
            const uint32_t base = smem_u32(smem + (size_t)s * stage_bytes);
            if (elect_one()) {
                const uint64_t wd = make_smem_desc(base, 16, 1024, kSwizzle128B), xd = make_smem_desc(base + kHalfTileBytes, 16, 1024, kSwizzle128B);
#pragma unroll
                for (uint32_t kk = 0; kk < 4; kk++) {
                    const uint32_t accumulate = (kb != kb0 || kk != 0) ? 1u : 0u;
                    if constexpr (DT == CLPK_DT_I8)
                        mma_i8_ss(tmem, wd + 2 * kk, xd + 2 * kk, idesc, accumulate);
                    else
                        mma_f16_ss(tmem, wd + 2 * kk, xd + 2 * kk, idesc, accumulate);
                }
                tc_commit(&sh->empty[s]);
            }
            __syncwarp();
            if (++s == p.stages) {
                s = 0;
                parity ^= 1;
            }
        }
        if (ok && elect_one())
            tc_commit(&sh->done);
        __syncwarp();
    }
    __syncwarp();
    // ---------------- partial sums -> shared memory, [token][128 rows] ----------------
    // All instructions have retired, hence all loads have landed: the ring is free.  A wait that ran out leaves sums that are
    // wrong, and a status that says so; every CTA still comes to the barriers below.
    if (!warp_wait(&sh->done, 0) && lane == 0)
        atomicCAS(p.status, 0u, 0x313u);
    tc_fence_after_sync();
    float *sums = reinterpret_cast<float *>(smem);
    for (uint32_t c = 0; c < p.m; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + ((uint32_t)warp * 32 << 16) + c, v);
        tmem_ld_wait();
#pragma unroll
        for (uint32_t i = 0; i < 16; i++)
            sums[(c + i) * kFewRows + threadIdx.x] = __uint_as_float(v[i]);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (p.splits > 1)
        cluster_sync();
    if (warp == 1)
        tmem_dealloc<1>(tmem, p.tmem_cols);

    // ---------------- the tokens of this CTA's turn: add over the cluster, finish, store ----------------
    constexpr uint32_t kPerLane = kTileCols / 32;
    const uint32_t col = tile * kTileCols + lane * kPerLane, left = col < p.n ? p.n - col : 0;
    float b_scale[kPerLane], u_scale[kPerLane];
#pragma unroll
    for (uint32_t i = 0; i < kPerLane; i++) {
        b_scale[i] = u_scale[i] = 0.0f;
        if (DT == CLPK_DT_I8 && i < left) {
            b_scale[i] = p.b_scale[col + i];
            if constexpr (FORM == kGated)
                u_scale[i] = p.u_scale[col + i];
            else if (p.bias)
                u_scale[i] = bias_at(p.bias, p.out, col + i);
        }
    }
    auto total = [&](uint32_t token, uint32_t first, float (&v)[kPerLane]) {
        uint32_t sum[kPerLane];
        for (uint32_t src = 0; src < p.splits; src++) {
            const uint32_t at = cluster_addr(sums + token * kFewRows + first + lane * kPerLane, src);
            uint32_t e[kPerLane];
            if constexpr (kPerLane == 4)
                asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(e[0]), "=r"(e[1]), "=r"(e[2]), "=r"(e[3]) : "r"(at) : "memory");
            else
                asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=r"(e[0]), "=r"(e[1]) : "r"(at) : "memory");
#pragma unroll
            for (uint32_t i = 0; i < kPerLane; i++) {
                if (src == 0)
                    sum[i] = e[i];
                else if constexpr (DT == CLPK_DT_I8)
                    sum[i] += e[i];
                else
                    sum[i] = __float_as_uint(__uint_as_float(sum[i]) + __uint_as_float(e[i]));
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kPerLane; i++)
            v[i] = DT == CLPK_DT_I8 ? (float)(int32_t)sum[i] : __uint_as_float(sum[i]);
    };
    for (uint32_t token = split * 4 + warp; token < p.m; token += 4 * p.splits) {
        const uint64_t at = token * p.ldc + col;
        float v[kPerLane], u[kPerLane];
        total(token, 0, v);
        if constexpr (FORM == kGated)
            total(token, 64, u);
        if constexpr (DT == CLPK_DT_I8) {
            const float row_scale = p.a_scale[token];
#pragma unroll
            for (uint32_t i = 0; i < kPerLane; i++) {
                v[i] = v[i] * row_scale * b_scale[i];
                if constexpr (FORM == kGated)
                    u[i] = u[i] * row_scale * u_scale[i];
                else if (p.bias)
                    v[i] += u_scale[i];
            }
        }
        if constexpr (FORM == kGated) {
            if (p.g) {
                few_store(p.g, p.out, at, left, v);
                few_store(p.u, p.out, at, left, u);
            }
#pragma unroll
            for (uint32_t i = 0; i < kPerLane; i++)
                v[i] = activate_by(p.activation, v[i]) * u[i];
        }
        few_store(p.c, p.out, at, left, v);
    }
    // nobody's sums go away while another CTA reads them
    if (p.splits > 1)
        cluster_sync();
}
