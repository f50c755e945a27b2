// Products of 8-bit rows with an 8-bit weight on tcgen05 / TMEM / TMA:
//
//     y[m, n] = a_scale[m] * b_scale[n] * sum_k a[m, k] b[n, k]          a [M, K], b [N, K] codes, K contiguous
//
// int8 codes (kind::i8, sums exact in 32-bit integers) or e4m3 codes (kind::f8f6f4, sums in f32); the scales and the one rounding of y are the
// epilogue.  A K block is 128 bytes of every row, so stages, swizzle and descriptors are those of the f16 product at twice the operations a byte.
#include "sm100_ptx.cuh"
#include "common.cuh"

namespace {
using namespace sm100;

constexpr int QM = 128, QK = 128;                                // tile rows and bytes of a K block
constexpr uint32_t Q_A_BYTES = QM * QK;
constexpr int Q_EPI_WG = 2;
constexpr int Q_THREADS = 64 + 128 * Q_EPI_WG;

template <int BN>
struct QShape {
    static constexpr uint32_t B_BYTES = BN * QK;
    static constexpr int STAGES = 4;
    static constexpr uint32_t RING = STAGES * (Q_A_BYTES + B_BYTES);
    static constexpr uint32_t SMEM = RING + 256;
    static constexpr int FULL = 0, EMPTY = STAGES, ACC_FULL = 2 * STAGES, ACC_EMPTY = ACC_FULL + 2, COUNT = ACC_EMPTY + 2;
};

struct GemmQ8Params {
    void* c;
    const float* sa; const float* sb;
    long long ldc;
    int M, N, K;
    int vec;                                                     // rows of c on 16-byte boundaries
    unsigned int* err;
};

template <bool I8>
__host__ __device__ constexpr uint32_t idesc_q8(int M, int N) {
    return (I8 ? (2u << 4) | (1u << 7) | (1u << 10) : 1u << 4)   // i8: sums s32, both signed; e4m3: sums f32, formats 0
           | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
template <bool I8>
__device__ __forceinline__ void umma_q8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (I8)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

template <bool I8>
__device__ __forceinline__ float sum_of(uint32_t r) { return I8 ? __int2float_rn((int)r) : __uint_as_float(r); }

// Barriers and tensor memory: nothing of global memory (see started()).
template <int BN>
__device__ __forceinline__ void gemm_q8_prologue(const void* tmap_a, const void* tmap_b) {
    using S = QShape<BN>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(bars + S::COUNT);
    if (threadIdx.x == 0) {
        tmem_base_s[1] = 0;                                      // the abort flag
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&bars[S::FULL + s], 1); mbar_init(&bars[S::EMPTY + s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&bars[S::ACC_FULL + s], 1); mbar_init(&bars[S::ACC_EMPTY + s], 4 * Q_EPI_WG); }
        fence_barrier_init();
        tma_prefetch_desc(tmap_a); tma_prefetch_desc(tmap_b);
    }
    if (uniform((int)threadIdx.x / 32) == 1) { tmem_alloc(tmem_base_s, 512); tmem_relinquish(); }
}

template <bool I8, typename T, int BN>
__global__ void __launch_bounds__(Q_THREADS, 1)
gemm_q8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const GemmQ8Params p) {
    gemm_q8_prologue<BN>(&tmap_a, &tmap_b);
    chain_wait();
    using S = QShape<BN>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t* sA = smem;
    uint8_t* sB = smem + S::STAGES * Q_A_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(bars + S::COUNT);
    volatile uint32_t* abort_s = tmem_base_s + 1;
    uint32_t* skip_s = tmem_base_s + 2;

    const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
    const int tiles_m = (p.M + QM - 1) / QM, tiles_n = (p.N + BN - 1) / BN, n_tiles = tiles_m * tiles_n;
    const int kbs = (p.K + QK - 1) / QK;
    if (!started(smem, skip_s, p.err, DEERS_KERR_GEMM | 0x60)) {
        if (warp == 1) tmem_dealloc(*tmem_base_s, 512);
        return;
    }
    const uint32_t tmem = (uint32_t)uniform((int)*tmem_base_s);
    WaitState ws{abort_s, p.err};

    if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < n_tiles; t += gridDim.x) {
                const int m0 = t % tiles_m * QM, n0 = t / tiles_m * BN;
                for (int kb = 0; kb < kbs; ++kb, ++g) {
                    const uint32_t s = g % S::STAGES;
                    if (!mbar_wait(ws, &bars[S::EMPTY + s], ((g / S::STAGES) & 1u) ^ 1u, DEERS_KERR_GEMM | 0x61)) { ok = false; break; }
                    mbar_arrive_expect_tx(&bars[S::FULL + s], Q_A_BYTES + S::B_BYTES);
                    tma_load_4d(sA + s * Q_A_BYTES, &tmap_a, &bars[S::FULL + s], kb * QK, m0, 0, 0);
                    tma_load_4d(sB + s * S::B_BYTES, &tmap_b, &bars[S::FULL + s], kb * QK, n0, 0, 0);
                }
            }
        }
        __syncwarp();
        chain_next();
    } else if (warp == 1) {
        constexpr uint32_t IDESC = idesc_q8<I8>(QM, BN);
        const uint64_t a0 = desc_kmajor((uint32_t)uniform((int)smem_u32(sA)), 0, 0), b0 = desc_kmajor((uint32_t)uniform((int)smem_u32(sB)), 0, 0);
        uint32_t g = 0;
        int n = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < n_tiles; t += gridDim.x, ++n) {
            const uint32_t buf = (uint32_t)n & 1u;
            if (!mbar_wait_warp(ws, &bars[S::ACC_EMPTY + buf], (((uint32_t)n >> 1) & 1u) ^ 1u, DEERS_KERR_GEMM | 0x62)) break;
            tc_fence_after_sync();
            for (int kb = 0; kb < kbs; ++kb, ++g) {
                const uint32_t s = g % S::STAGES;
                if (!mbar_wait_warp(ws, &bars[S::FULL + s], (g / S::STAGES) & 1u, DEERS_KERR_GEMM | 0x63)) { ok = false; break; }
                tc_fence_after_sync();
                const uint64_t a = a0 + (uint64_t)s * (Q_A_BYTES >> 4), b = b0 + (uint64_t)s * (S::B_BYTES >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)                // 32 bytes of K a product
                        umma_q8<I8>(tmem + buf * 256u, a + kmajor_step(ks, 0), b + kmajor_step(ks, 0), IDESC, kb > 0 || ks > 0);
                    umma_commit(&bars[S::EMPTY + s]);
                    if (kb == kbs - 1) umma_commit(&bars[S::ACC_FULL + buf]);
                }
                __syncwarp();
            }
        }
    } else {
        constexpr int PER = 16 / (int)sizeof(T), CH = 8 * PER, SHARE = BN / Q_EPI_WG;
        static_assert(SHARE % CH == 0, "whole chunks");
        const int lane_base = (warp & 3) * 32, share0 = ((warp - 2) >> 2) * SHARE;
        const uint32_t t_lane = (uint32_t)lane_base << 16;
        int n = 0;
        for (int t = blockIdx.x; t < n_tiles; t += gridDim.x, ++n) {
            const int m0 = t % tiles_m * QM, n0 = t / tiles_m * BN;
            const uint32_t buf = (uint32_t)n & 1u;
            if (!__all_sync(0xffffffffu, mbar_wait(ws, &bars[S::ACC_FULL + buf], ((uint32_t)n >> 1) & 1u, DEERS_KERR_GEMM | 0x64))) break;
            tc_fence_after_sync();
            const float sa = m0 + lane_base + lane < p.M ? p.sa[m0 + lane_base + lane] : 0.f;
            const int row0 = m0 + lane_base + (lane & ~7);
#pragma unroll 1
            for (int c0 = share0; c0 < share0 + SHARE; c0 += CH) {
                uint32_t r[CH];
                uint4 pc[8];
#pragma unroll
                for (int c = 0; c < CH; c += 32) tmem_ld_x32(tmem + buf * 256u + t_lane + c0 + c, *reinterpret_cast<uint32_t(*)[32]>(&r[c]));
                tmem_wait_ld();
                if (c0 == share0 + SHARE - CH) {
                    tc_fence_before_sync();
                    mbar_arrive_warp(&bars[S::ACC_EMPTY + buf]);
                }
                if (n0 + c0 >= p.N) continue;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    float v[PER];
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        const int col = n0 + c0 + q * PER + e;
                        v[e] = sum_of<I8>(r[q * PER + e]) * sa * (col < p.N ? p.sb[col] : 0.f);
                    }
                    if constexpr (PER == 8) pc[q] = make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
                    else pc[q] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                }
                transpose_pieces<8>(pc, (uint32_t)lane);
                const int col = n0 + c0 + (lane & 7) * PER;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int row = row0 + c;
                    if (row >= p.M || col >= p.N) continue;
                    T* to = static_cast<T*>(p.c) + (long long)row * p.ldc + col;
                    if (p.vec && col + PER <= p.N) {
                        *reinterpret_cast<uint4*>(to) = pc[c];
                    } else {
                        const T* v = reinterpret_cast<const T*>(&pc[c]);
#pragma unroll
                        for (int e = 0; e < PER; ++e)
                            if (col + e < p.N) to[e] = v[e];
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, 512);
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Map over [rows][inner] bytes, rows ld bytes apart: boxes of 128 bytes by box_rows rows, 128-byte swizzle, zeros outside.
int tmap_bytes(deers_ctx* ctx, CUtensorMap* out, const void* base, long long rows, long long inner, long long ld, int box_rows) {
    if (!ctx->encode_tiled) {
        snprintf(ctx->last_error, sizeof(ctx->last_error), "cuTensorMapEncodeTiled not available");
        return DEERS_ERR_CUDA;
    }
    const cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)rows, 1, 1};
    const cuuint64_t far = (cuuint64_t)ld * (cuuint64_t)rows;
    const cuuint64_t strides[3] = {(cuuint64_t)ld, far, far};
    const cuuint32_t box[4] = {(cuuint32_t)QK, (cuuint32_t)box_rows, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = ((EncodeTiled)ctx->encode_tiled)(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, one,
                                                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        snprintf(ctx->last_error, sizeof(ctx->last_error), "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
        return DEERS_ERR_LAYOUT;
    }
    return DEERS_OK;
}

template <bool I8, typename T>
int gemm_q8_launch(deers_ctx* ctx, const GemmQ8Params& p, const void* a, long long lda, const void* b, long long ldb) {
    constexpr int BN = 256;
    using S = QShape<BN>;
    CUtensorMap ta, tb;
    int rc = tmap_bytes(ctx, &ta, a, p.M, p.K, lda, QM);
    if (!rc) rc = tmap_bytes(ctx, &tb, b, p.N, p.K, ldb, BN);
    if (rc) return rc;
    const long long tiles = (long long)((p.M + QM - 1) / QM) * ((p.N + BN - 1) / BN);
    const unsigned grid = (unsigned)(tiles < ctx->sm_count ? tiles : ctx->sm_count);
    DEERS_SMEM_ONCE(ctx, (gemm_q8_kernel<I8, T, BN>), S::SMEM);
    KernelTimerScope ts(ctx, DEERS_K_GEMM);
    DEERS_CUDA_TRY(ctx, launch_chained(ctx, gemm_q8_kernel<I8, T, BN>, grid, Q_THREADS, S::SMEM, 1, ta, tb, p));
    return DEERS_OK;
}

}  // namespace

extern "C" int deers_b200_gemm_q8(deers_ctx* ctx, int32_t M, int32_t N, int32_t K, int32_t code, const void* a, int64_t lda, const float* a_scale,
                                  const void* b, int64_t ldb, const float* b_scale, int32_t out_dtype, void* c, int64_t ldc) {
    if (!ctx) return DEERS_ERR_NULL;
    if (code != DEERS_I8 && code != DEERS_E4M3) return DEERS_ERR_DTYPE;
    if (out_dtype != DEERS_F16 && out_dtype != DEERS_F32) return DEERS_ERR_DTYPE;
    if (M < 0 || N < 1 || K < 1) return DEERS_ERR_SHAPE;
    if (code == DEERS_I8 && K > 131072) return DEERS_ERR_UNSUPPORTED;        // 2^31 / 128^2: sums stay whole numbers of 32 bits
    if (M == 0) return DEERS_OK;
    if (!a || !b || !c || !a_scale || !b_scale) return DEERS_ERR_NULL;
    const uintptr_t es = out_dtype == DEERS_F16 ? 2 : 4;
    if (((uintptr_t)a | (uintptr_t)b) & 15u || (lda | ldb) & 15 || lda < K || ldb < K || ldc < N) return DEERS_ERR_LAYOUT;
    if (((uintptr_t)a_scale | (uintptr_t)b_scale) & 3u || (uintptr_t)c & (es - 1)) return DEERS_ERR_LAYOUT;
    DEERS_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    GemmQ8Params p;
    p.c = c; p.sa = a_scale; p.sb = b_scale; p.ldc = ldc; p.M = M; p.N = N; p.K = K; p.err = ctx->dev_err;
    p.vec = ((uintptr_t)c & 15u) == 0 && (ldc * (int64_t)es & 15) == 0;
    const auto go = code == DEERS_I8 ? (out_dtype == DEERS_F16 ? gemm_q8_launch<true, __half> : gemm_q8_launch<true, float>)
                                     : (out_dtype == DEERS_F16 ? gemm_q8_launch<false, __half> : gemm_q8_launch<false, float>);
    const int rc = go(ctx, p, a, lda, b, ldb);
    if (rc) return rc;
    ctx->launches += 1;
    DEERS_CUDA_TRY(ctx, cudaGetLastError());
    return DEERS_OK;
}
