// Products of 8-bit rows with an 8-bit weight on tcgen05 / TMEM / TMA:
//
//     y[m, n] = (a_scale[m] * b_scale[n]) * sum_k a[m, k] b[n, k]          a [M, K], b [N, K] codes, K contiguous
//
// int8 codes (kind::i8, sums exact in 32-bit integers) or e4m3 codes (kind::f8f6f4, sums in f32, cut off); the scales and the rounding of y are the
// epilogue.  The scales meet first: large rows and small weights bring one another back, where a sum times one of them could leave f32.
// A K block is 128 bytes of every row, so stages, swizzle and descriptors are those of the f16 product at twice the operations a byte.
// Large products go to persistent CTAs or pairs of them (8192 x 4096 x 4096 int8 90 us, 3050 TOP/s: 0.93 of twice the measured bf16 peak, e4m3 97 to 99;
// without a pause between calls, under the power cap, int8 104), products with few tiles to clusters that share a tile's K, a step's few tokens to tiles
// that have the weight's rows for rows (64 x 4096 x 12288 15 us).
// What bounds them: large ones the tensor pipe; steps the weight's bytes (here 8 us) and, before and behind them, 2 us to the first K block and 2 to 4 from the
// last product to the end.
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

#include <cooperative_groups.h>

namespace {
using namespace sm100;

constexpr int QM = 128, QK = 128;                                // tile rows and bytes of a K block
constexpr uint32_t Q_A_BYTES = QM * QK;
constexpr int Q_EPI_WG = 2;
constexpr int Q_THREADS = 64 + 128 * Q_EPI_WG;

// Tiles of 128 x BN by one CTA, or of 256 x BN by a pair of CTAs on two SMs, each with half of the rows and half of B's columns.
template <int BN, bool PAIR>
struct QShape {
    static constexpr uint32_t B_BYTES = (PAIR ? BN / 2 : BN) * QK;
    static constexpr int STAGES = PAIR ? 6 : 4;
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
    int kb_chunk;                                                // K blocks of a part
    unsigned int* err;
};

template <bool I8>
__host__ __device__ constexpr uint32_t idesc_q8(int M, int N) {
    return (I8 ? (2u << 4) | (1u << 7) | (1u << 10) : 1u << 4)   // i8: sums s32, both signed; e4m3: sums f32, formats 0
           | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
#define DEERS_UMMA_Q8(GROUP, KIND)                                                                                                             \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" \
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory")
template <bool I8, bool PAIR = false>
__device__ __forceinline__ void umma_q8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR) {
        if constexpr (I8) DEERS_UMMA_Q8("2", "i8");
        else DEERS_UMMA_Q8("2", "f8f6f4");
    } else {
        if constexpr (I8) DEERS_UMMA_Q8("1", "i8");
        else DEERS_UMMA_Q8("1", "f8f6f4");
    }
}
#undef DEERS_UMMA_Q8

template <bool I8>
__device__ __forceinline__ float sum_of(uint32_t r) { return I8 ? __int2float_rn((int)r) : __uint_as_float(r); }

// 16 bytes of a row of c.
template <typename T>
__device__ __forceinline__ uint4 packed(const float* v) {
    if constexpr (sizeof(T) == 2) return make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
    else return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
// They go to column col on, or what of them is inside.
template <typename T>
__device__ __forceinline__ void store_piece(const GemmQ8Params& p, int row, int col, const uint4& w) {
    constexpr int PER = 16 / (int)sizeof(T);
    T* to = static_cast<T*>(p.c) + (long long)row * p.ldc + col;
    if (p.vec && col + PER <= p.N) {
        *reinterpret_cast<uint4*>(to) = w;
    } else {
        const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int e = 0; e < PER; ++e)
            if (col + e < p.N) to[e] = x[e];
    }
}

// Barriers and tensor memory: nothing of global memory (see started()).
template <int BN, bool PAIR>
__device__ __forceinline__ void gemm_q8_prologue(const void* tmap_a, const void* tmap_b) {
    using S = QShape<BN, PAIR>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(bars + S::COUNT);
    if (threadIdx.x == 0) {
        tmem_base_s[1] = 0;                                      // the abort flag
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&bars[S::FULL + s], 1); mbar_init(&bars[S::EMPTY + s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&bars[S::ACC_FULL + s], 1); mbar_init(&bars[S::ACC_EMPTY + s], (PAIR ? 8 : 4) * Q_EPI_WG); }
        fence_barrier_init();
        tma_prefetch_desc(tmap_a); tma_prefetch_desc(tmap_b);
    }
    if (uniform((int)threadIdx.x / 32) == 1) {
        if (PAIR) { tmem_alloc_pair(tmem_base_s, 512); tmem_relinquish_pair(); }
        else { tmem_alloc(tmem_base_s, 512); tmem_relinquish(); }
    }
}

// Persistent: warp 0 streams K blocks of both operands through a ring, warp 1 issues their products into one of two accumulators, the other warps take
// a finished one out, scale, round and store it while the next one fills.  Of a pair the first CTA issues for both: B is read from both shared memories, which
// a CTA alone (187 bytes a cycle of the 128 it has) waits for.
template <bool I8, typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(Q_THREADS, 1)
gemm_q8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const GemmQ8Params p) {
    gemm_q8_prologue<BN, PAIR>(&tmap_a, &tmap_b);
    chain_wait();
    namespace cg = cooperative_groups;
    using S = QShape<BN, PAIR>;
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int TM = PAIR ? 2 * QM : QM, HALF_B = PAIR ? BN / 2 : BN;
    uint8_t* sA = smem;
    uint8_t* sB = smem + S::STAGES * Q_A_BYTES;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(bars + S::COUNT);
    volatile uint32_t* abort_s = tmem_base_s + 1;
    uint32_t* skip_s = tmem_base_s + 2;

    const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
    const int tiles_m = (p.M + TM - 1) / TM, tiles_n = (p.N + BN - 1) / BN, n_tiles = tiles_m * tiles_n;
    const int kbs = (p.K + QK - 1) / QK;
    const int half = PAIR ? (int)cg::this_cluster().block_rank() : 0;
    const int t0 = PAIR ? (int)blockIdx.x / 2 : (int)blockIdx.x, t_step = PAIR ? (int)gridDim.x / 2 : (int)gridDim.x;
    bool skip = !started(smem, skip_s, p.err, DEERS_KERR_GEMM | 0x60);
    if constexpr (PAIR) {
        cg::this_cluster().sync();                               // both have their barriers, and both go on or neither
        skip = skip || *cg::this_cluster().map_shared_rank(skip_s, half ^ 1) != 0;
    }
    const uint32_t tmem = (uint32_t)uniform((int)*tmem_base_s);
    WaitState ws{abort_s, p.err};

    if (skip) {
    } else if (warp == 0) {
        if (lane == 0) {
            uint32_t g = 0;
            bool ok = true;
            for (int t = t0; ok && t < n_tiles; t += t_step) {
                const int m0 = t % tiles_m * TM + half * QM, n0 = t / tiles_m * BN + half * HALF_B;
                for (int kb = 0; kb < kbs; ++kb, ++g) {
                    const uint32_t s = g % S::STAGES;
                    if (!mbar_wait(ws, &bars[S::EMPTY + s], ((g / S::STAGES) & 1u) ^ 1u, DEERS_KERR_GEMM | 0x61)) { ok = false; break; }
                    // (a pair's stage is announced at its first CTA, for the bytes of both)
                    constexpr uint32_t BYTES = Q_A_BYTES + S::B_BYTES;
                    if (half == 0) mbar_arrive_expect_tx(&bars[S::FULL + s], PAIR ? 2 * BYTES : BYTES);
                    if constexpr (PAIR) {
                        const uint32_t full = cluster_addr(&bars[S::FULL + s], 0);
                        tma_load_4d_pair(sA + s * Q_A_BYTES, &tmap_a, full, kb * QK, m0, 0, 0);
                        tma_load_4d_pair(sB + s * S::B_BYTES, &tmap_b, full, kb * QK, n0, 0, 0);
                    } else {
                        tma_load_4d(sA + s * Q_A_BYTES, &tmap_a, &bars[S::FULL + s], kb * QK, m0, 0, 0);
                        tma_load_4d(sB + s * S::B_BYTES, &tmap_b, &bars[S::FULL + s], kb * QK, n0, 0, 0);
                    }
                }
            }
        }
        __syncwarp();
        chain_next();
    } else if (warp == 1) {
        if (half == 0) {
            constexpr uint32_t IDESC = idesc_q8<I8>(TM, BN);
            const auto commit = [&](uint64_t* bar) {
                if constexpr (PAIR) umma_commit_pair(bar, 3u);
                else umma_commit(bar);
            };
            const uint64_t a0 = desc_kmajor((uint32_t)uniform((int)smem_u32(sA)), 0, 0), b0 = desc_kmajor((uint32_t)uniform((int)smem_u32(sB)), 0, 0);
            uint32_t g = 0;
            int n = 0;
            bool ok = true;
            for (int t = t0; ok && t < n_tiles; t += t_step, ++n) {
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
                        for (int ks = 0; ks < 4; ++ks)            // 32 bytes of K a product
                            umma_q8<I8, PAIR>(tmem + buf * 256u, a + kmajor_step(ks, 0), b + kmajor_step(ks, 0), IDESC, kb > 0 || ks > 0);
                        commit(&bars[S::EMPTY + s]);
                        if (kb == kbs - 1) commit(&bars[S::ACC_FULL + buf]);
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        constexpr int PER = 16 / (int)sizeof(T), CH = 8 * PER, SHARE = BN / Q_EPI_WG;
        static_assert(SHARE % CH == 0, "whole chunks");
        const int lane_base = (warp & 3) * 32, share0 = ((warp - 2) >> 2) * SHARE;
        const uint32_t t_lane = (uint32_t)lane_base << 16;
        int n = 0;
        for (int t = t0; t < n_tiles; t += t_step, ++n) {
            const int m0 = t % tiles_m * TM + half * QM, n0 = t / tiles_m * BN;
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
                    if constexpr (PAIR) mbar_arrive_cluster_warp(cluster_addr(&bars[S::ACC_EMPTY + buf], 0));
                    else mbar_arrive_warp(&bars[S::ACC_EMPTY + buf]);
                }
                if (n0 + c0 >= p.N) continue;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    float v[PER];
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        const int col = n0 + c0 + q * PER + e;
                        v[e] = sum_of<I8>(r[q * PER + e]) * (sa * (col < p.N ? p.sb[col] : 0.f));
                    }
                    pc[q] = packed<T>(v);
                }
                transpose_pieces<8>(pc, (uint32_t)lane);
                const int col = n0 + c0 + (lane & 7) * PER;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int row = row0 + c;
                    if (row < p.M && col < p.N) store_piece<T>(p, row, col, pc[c]);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) cg::this_cluster().sync();               // nobody leaves while its peer still reads its memory or arrives at its barriers
    if (warp == 1) {
        if constexpr (PAIR) tmem_dealloc_pair(tmem, 512);
        else tmem_dealloc(tmem, 512);
    }
}

// ---- products with few tiles: a tile per cluster, whose CTAs take a share of K each
// SWAP: the weight's rows are the 128 rows of the tensor core's tile and the BN columns are rows of a, so that a step of few tokens fills the tile and
// moves each byte of the weight once.  Each CTA of a cluster owns a share of the tensor core's rows.  When all have their sums, every thread sends
// those of its row to the owner's shared memory (over the ring), which adds them in the order of their K ranges: no workspace, int8 sums
// stay whole numbers, and nobody waits for a remote load.  (Loads of parked tiles took 3.8 us of 128 x 128 values in four parts.)
constexpr int QS_EPI_WG = 2, QS_THREADS = 64 + 128 * QS_EPI_WG;  // warpgroups that share a tile's columns
constexpr int QS_MAX_PARTS = 8;
template <int BN, bool SWAP>
struct SplitShape {
    static constexpr uint32_t B_BYTES = BN * QK, STAGE = Q_A_BYTES + B_BYTES;
    static constexpr int STAGES = BN == 256 ? 4 : BN == 128 ? 3 : BN == 64 ? 4 : BN == 32 ? 5 : 6;      // two CTAs an SM but for 256
    static constexpr uint32_t RING = STAGES * STAGE, SCALES = RING + 256, SMEM = SCALES + 4 * (QM + BN);    // scales of the tile's rows and columns
    static constexpr int ROWS = SWAP ? BN : QM, COLS = SWAP ? QM : BN;                                  // of c
    static constexpr int FULL = 0, EMPTY = STAGES, DONE = 2 * STAGES, COUNT = DONE + 1;
    static constexpr uint32_t TMEM = BN < 32 ? 32 : BN;
    static constexpr int LD = BN + 4;                                                                   // !SWAP: sums of a row, as they are sent
    static_assert((uint32_t)(SWAP ? 7 * 24 * BN : (QM + QS_MAX_PARTS) * LD) * 4 <= RING, "what is sent fits over the ring (seven shares of 24 rows are the most)");
    static_assert(COUNT * 8 + 12 + 4 * QS_MAX_PARTS <= 256, "barriers and flags");
};
// Rows of the tensor core's tile that a CTA of `parts` owns (SWAP: whole 16-byte pieces of c).
template <bool SWAP>
__host__ __device__ constexpr int split_share(int parts) { return SWAP ? ((QM + parts - 1) / parts + 7) / 8 * 8 : (QM + parts - 1) / parts; }
__device__ __forceinline__ void send(uint32_t to, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(v) : "memory"); }
__device__ __forceinline__ void send(uint32_t to, const uint4& v) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <int BN, bool SWAP>
__device__ __forceinline__ void split_prologue(const void* tmap_a, const void* tmap_b) {
    using S = SplitShape<BN, SWAP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(bars + S::COUNT);
    if (threadIdx.x == 0) {
        tmem_base_s[1] = 0;                                      // the abort flag
        for (int s = 0; s < S::STAGES; ++s) { mbar_init(&bars[S::FULL + s], 1); mbar_init(&bars[S::EMPTY + s], 1); }
        mbar_init(&bars[S::DONE], 1);
        fence_barrier_init();
        tma_prefetch_desc(tmap_a); tma_prefetch_desc(tmap_b);
    }
    if (uniform((int)threadIdx.x / 32) == 1) { tmem_alloc(tmem_base_s, S::TMEM); tmem_relinquish(); }
}

template <bool I8, typename T, int BN, bool SWAP>
__global__ void __launch_bounds__(QS_THREADS)
gemm_q8_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const GemmQ8Params p) {
    split_prologue<BN, SWAP>(&tmap_a, &tmap_b);
    chain_wait();
    namespace cg = cooperative_groups;
    using S = SplitShape<BN, SWAP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::RING);
    uint32_t* tmem_base_s = reinterpret_cast<uint32_t*>(bars + S::COUNT);
    volatile uint32_t* abort_s = tmem_base_s + 1;
    uint32_t* skip_s = tmem_base_s + 2;
    uint32_t* have_s = tmem_base_s + 3;                          // [part]: its sums are there

    const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
    const cg::cluster_group cluster = cg::this_cluster();
    const int part = (int)cluster.block_rank(), parts = (int)cluster.num_blocks(), tile = (int)blockIdx.x / parts;
    const int tiles_a = ((SWAP ? p.N : p.M) + QM - 1) / QM;
    const int a0 = tile % tiles_a * QM, b0 = tile / tiles_a * BN;               // first row of either operand
    const int kb0 = part * p.kb_chunk, kb1 = min((p.K + QK - 1) / QK, kb0 + p.kb_chunk);
    const int m0 = SWAP ? b0 : a0, n0 = SWAP ? a0 : b0;
    float* scales = reinterpret_cast<float*>(smem + S::SCALES);
    const bool skip = !started(smem, skip_s, p.err, DEERS_KERR_GEMM | 0x68);    // (a CTA of a cluster stays: its peers read its shared memory)
    const uint32_t tmem = (uint32_t)uniform((int)*tmem_base_s);
    WaitState ws{abort_s, p.err};
    if (parts > 1) cluster.barrier_arrive();                     // (waited for before anybody writes to another's shared memory)
    bool done = false;                                           // (warps 2 on) this CTA's sums are there
    if (skip) {
    } else if (warp == 0) {
        if (lane == 0) {
            int kb = kb0 + tile % (kb1 - kb0);
            for (int g = 0; g < kb1 - kb0; ++g, kb = kb + 1 == kb1 ? kb0 : kb + 1) {
                const uint32_t s = g % S::STAGES;
                if (!mbar_wait(ws, &bars[S::EMPTY + s], ((g / S::STAGES) & 1u) ^ 1u, DEERS_KERR_GEMM | 0x69)) break;
                mbar_arrive_expect_tx(&bars[S::FULL + s], S::STAGE);
                tma_load_4d(smem + s * S::STAGE, &tmap_a, &bars[S::FULL + s], kb * QK, a0, 0, 0);
                tma_load_4d(smem + s * S::STAGE + Q_A_BYTES, &tmap_b, &bars[S::FULL + s], kb * QK, b0, 0, 0);
            }
        }
        __syncwarp();
        chain_next();
    } else if (warp == 1) {
        constexpr uint32_t IDESC = idesc_q8<I8>(QM, BN);
        const uint32_t at = (uint32_t)uniform((int)smem_u32(smem));
        const uint64_t da = desc_kmajor(at, 0, 0), db = desc_kmajor(at + Q_A_BYTES, 0, 0);
        for (int kb = kb0, g = 0; kb < kb1; ++kb, ++g) {
            const uint32_t s = g % S::STAGES;
            if (!mbar_wait_warp(ws, &bars[S::FULL + s], (g / S::STAGES) & 1u, DEERS_KERR_GEMM | 0x6a)) break;
            tc_fence_after_sync();
            const uint64_t a = da + (uint64_t)s * (S::STAGE >> 4), b = db + (uint64_t)s * (S::STAGE >> 4);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) umma_q8<I8>(tmem, a + kmajor_step(ks, 0), b + kmajor_step(ks, 0), IDESC, g > 0 || ks > 0);
                umma_commit(&bars[S::EMPTY + s]);
                if (kb == kb1 - 1) umma_commit(&bars[S::DONE]);
            }
            __syncwarp();
        }
    } else {
        // the scales, while the products run
        for (int i = (int)threadIdx.x - 64; i < S::ROWS + S::COLS; i += 128 * QS_EPI_WG) {
            const bool of_row = i < S::ROWS;
            const int at = of_row ? m0 + i : n0 + i - S::ROWS;
            scales[i] = at < (of_row ? p.M : p.N) ? (of_row ? p.sa : p.sb)[at] : 0.f;
        }
        done = __all_sync(0xffffffffu, mbar_wait(ws, &bars[S::DONE], 0, DEERS_KERR_GEMM | 0x6b));
        tc_fence_after_sync();
    }
    __syncwarp();
    if (parts > 1) cluster.barrier_wait();
    if (warp == 2 && lane < parts) *(parts > 1 ? cluster.map_shared_rank(have_s + part, lane) : have_s) = done ? 1u : 0u;
    __syncwarp();
    const int rows = min(S::ROWS, p.M - m0), row = (warp & 3) * 32 + lane;      // (warps 2 on) this thread's row of the tensor core's tile
    const uint32_t t_lane = (uint32_t)((warp & 3) * 32) << 16;
    constexpr int CH = BN < 32 * QS_EPI_WG ? 16 : 32, PER = 16 / (int)sizeof(T);    // columns at a time; of a 16-byte piece of c
    const int ch0 = ((warp - 2) >> 2) * CH;                                     // warpgroups take turns
    const auto take = [&](int c0, uint32_t (&r)[CH]) {
        if constexpr (CH == 32) tmem_ld_x32(tmem + t_lane + c0, r);
        else tmem_ld_x16(tmem + t_lane + c0, r);
        tmem_wait_ld();
    };
    if (!SWAP && parts == 1) {
        __syncthreads();                                         // the scales are there
        if (done) {
            const float mine = scales[row];
#pragma unroll 1
            for (int c0 = ch0; c0 < BN; c0 += CH * QS_EPI_WG) {
                uint32_t r[CH];
                take(c0, r);
                constexpr int NP = CH / PER;                     // 4 or 8 pieces of a row, exchanged among as many lanes
                uint4 pc[NP];
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    float v[PER];
#pragma unroll
                    for (int e = 0; e < PER; ++e) v[e] = sum_of<I8>(r[q * PER + e]) * (mine * scales[S::ROWS + c0 + q * PER + e]);
                    pc[q] = packed<T>(v);
                }
                transpose_pieces<NP>(pc, (uint32_t)lane);
#pragma unroll
                for (int c = 0; c < NP; ++c) {
                    const int r1 = (row & ~(NP - 1)) + c;
                    if (r1 < rows) store_piece<T>(p, m0 + r1, n0 + c0 + (lane & (NP - 1)) * PER, pc[c]);
                }
            }
        }
    } else {
        const auto meet = [&]() {
            if (parts > 1) cluster.sync();
            else __syncthreads();
        };
        meet();                                                  // every ring has been read
        bool all = true;
        for (int z = 0; z < parts; ++z) all = all && have_s[z] != 0;
        // what is sent: SWAP [part][row of c][own columns of c], else [part][own row of c][LD]
        const int share = split_share<SWAP>(parts), of_part = SWAP ? rows * share : share * S::LD;
        const uint32_t* sent = reinterpret_cast<const uint32_t*>(smem);
        if (all && warp >= 2) {
            const int owner = row / share, at = row - owner * share;
            const uint32_t to = cluster_addr(smem, owner) + 4u * (uint32_t)(part * of_part + (SWAP ? at : at * S::LD));
#pragma unroll 1
            for (int c0 = ch0; c0 < (SWAP ? rows : BN); c0 += CH * QS_EPI_WG) {
                uint32_t r[CH];
                take(c0, r);
                if constexpr (SWAP) {
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        if (c0 + c < rows) send(to + 4u * (uint32_t)((c0 + c) * share), r[c]);
                } else {
#pragma unroll
                    for (int c = 0; c < CH; c += 4) send(to + 4u * (uint32_t)(c0 + c), make_uint4(r[c], r[c + 1], r[c + 2], r[c + 3]));
                }
            }
        }
        __syncwarp();
        meet();
        const int first = part * share, mine = min(share, QM - first);
        if (all && mine > 0) {
            // A thread adds up the same 16-byte piece of several rows of c.
            const int width = (SWAP ? mine : BN) / PER, c = (int)threadIdx.x % width * PER, step = QS_THREADS / width;
            const int r0 = SWAP ? 0 : first, col = SWAP ? first + c : c, ld = SWAP ? share : S::LD, n = SWAP ? rows : min(mine, rows - first);
            float sb[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) sb[e] = scales[S::ROWS + col + e];
#pragma unroll 2
            for (int r = (int)threadIdx.x / width; r < (threadIdx.x < step * width ? n : 0); r += step) {
                uint32_t v[PER];
#pragma unroll
                for (int e = 0; e < PER; e += 4) *reinterpret_cast<uint4*>(v + e) = *reinterpret_cast<const uint4*>(sent + r * ld + c + e);
                for (int z = 1; z < parts; ++z) {
                    uint32_t w[PER];
#pragma unroll
                    for (int e = 0; e < PER; e += 4) *reinterpret_cast<uint4*>(w + e) = *reinterpret_cast<const uint4*>(sent + z * of_part + r * ld + c + e);
#pragma unroll
                    for (int e = 0; e < PER; ++e) v[e] = I8 ? v[e] + w[e] : __float_as_uint(__uint_as_float(v[e]) + __uint_as_float(w[e]));
                }
                const float sa = scales[r0 + r];
                float f[PER];
#pragma unroll
                for (int e = 0; e < PER; ++e) f[e] = sum_of<I8>(v[e]) * (sa * sb[e]);
                if (n0 + col < p.N) store_piece<T>(p, m0 + r0 + r, n0 + col, packed<T>(f));
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, S::TMEM);
}

// Map over [rows][inner] bytes, rows ld bytes apart: boxes of 128 bytes by box_rows rows, 128-byte swizzle, zeros outside.
int tmap_bytes(deers_ctx* ctx, CUtensorMap* out, const void* base, long long rows, long long inner, long long ld, int box_rows) {
    const cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)rows, 1, 1}, far = (cuuint64_t)ld * (cuuint64_t)rows, strides[3] = {(cuuint64_t)ld, far, far};
    const cuuint32_t box[4] = {(cuuint32_t)QK, (cuuint32_t)box_rows, 1, 1};
    return make_tmap_bytes(ctx, out, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

struct GemmQ8Plan { int bn, parts; bool swap, split, pair; };

// The way with the least estimated time.  The estimate is in microseconds and was fitted to 2600 measured times (200 sizes of M 1 .. 8192, K 300 .. 16384,
// N 512 .. 12288; every way that is meant for them up to M 2048, the two persistent ones above); what it picks is 1.3 % slower than the best of those on
// average, 21 % at most.  Above M 2048 shares of K were not timed and are not picked, which leaves narrow products of long K behind: K 16384, N 512
// take 26 us at M 2048 and 43 at 2049 and 4096; 4096 x 8192 x 256 25 (6 by its bytes).  N below 512 was not swept.  Per K block a CTA needs 0.14 us with
// 16 columns to 0.37 with 256, a persistent one 0.45, a pair 0.33; a second CTA on an SM runs at 0.9 of the first's speed.  Adding up parts costs
// 1.6 and 0.03 a column, a pair's launch 2.6 more than a single CTA's.  1 x 768 x 2304 6.5 us by persistent CTAs, 4.0 swapped; 64 x 4096 x 12288 19.7 and 15.0;
// 64 x 11008 x 4096 36 and 14.3 in four parts; 333 x 2731 x 1001 29 and 10.1; 1024 x 768 x 2304 7.7 and 5.2; 8192 x 4096 x 4096 97.8, by pairs 89.4.
GemmQ8Plan plan_gemm_q8(int sms, int pairs, int M, int N, int K) {
    const int kbs = (K + QK - 1) / QK;
    const auto up = [](long long a, long long b) { return (a + b - 1) / b; };
    GemmQ8Plan best{256, 1, false, false, false};
    double least = 4.0 + (double)up(up(M, QM) * up(N, 256), sms) * (0.454 * kbs + 0.58);
    if (pairs > 0) {
        const double t = 6.6 + (double)up(up(M, 2 * QM) * up(N, 256), pairs) * (0.331 * kbs + 0.58);
        if (t < least) { least = t; best.pair = true; }
    }
    if (M > 2048) return best;
    static const double block[5] = {0.14, 0.30, 0.28, 0.33, 0.37};
    for (int w = 0; w < 5; ++w) {
        const int bn = 16 << w;
        for (int swap = 0; swap < 2; ++swap) {
            // what swapped tiles are for: as many columns as there are rows of a, 64 also several times; the others have 128 rows (and those of 128 columns
            // nothing over swapped ones)
            if (swap ? (bn > 64 || bn >= 2 * M + 32 || M > (bn < 64 ? bn : 4 * bn)) : (bn < 128 || M <= 64)) continue;
            const long long tiles = swap ? up(N, QM) * up(M, bn) : up(M, QM) * up(N, bn);
            for (int ask = 1; ask <= QS_MAX_PARTS; ++ask) {
                const int chunk = (int)up(kbs, ask), parts = (int)up(kbs, chunk);
                if (parts != ask) continue;
                double slots = bn == 256 ? sms : parts > 2 ? 1.04 * sms : 2.0 * sms;
                if (parts > 1) slots *= 0.88;                    // (clusters leave some SMs of a group empty)
                const double ctas = (double)tiles * parts, whole = ctas / slots, waves = (double)(long long)whole + (whole > (double)(long long)whole ? 1 : 0);
                const double load = ctas / sms / waves, rate = load <= 1 ? 1 : 1 + 1.19 * ((load < 2 ? load : 2) - 1);
                double t = 2.1 + waves * (chunk * block[w] * rate + 0.53 + 0.0088 * bn);
                if (parts > 1) t += 0.05 + 0.0285 * bn * (1.0 - 1.0 / parts) + 1.57 * waves;
                else if (swap) t += 0.021 * bn;
                if (t < least) { least = t; best = GemmQ8Plan{bn, parts, swap != 0, true, false}; }
            }
        }
    }
    return best;
}

int plan_gemm_q8(deers_ctx* ctx, int M, int N, int K, GemmQ8Plan* plan, int* pairs) {
    const int rc = gemm_f16_pairs(ctx, pairs);
    if (!rc) *plan = plan_gemm_q8(ctx->sm_count, *pairs, M, N, K);
    return rc;
}

template <bool I8, typename T, int BN, bool SWAP>
int gemm_q8_split(deers_ctx* ctx, GemmQ8Params p, const void* a, long long lda, const void* b, long long ldb, int parts) {
    using S = SplitShape<BN, SWAP>;
    CUtensorMap ta, tb;                                          // of the tensor core's rows and columns
    int rc = SWAP ? tmap_bytes(ctx, &ta, b, p.N, p.K, ldb, QM) : tmap_bytes(ctx, &ta, a, p.M, p.K, lda, QM);
    if (!rc) rc = SWAP ? tmap_bytes(ctx, &tb, a, p.M, p.K, lda, BN) : tmap_bytes(ctx, &tb, b, p.N, p.K, ldb, BN);
    if (rc) return rc;
    const long long tiles = (long long)((p.M + S::ROWS - 1) / S::ROWS) * ((p.N + S::COLS - 1) / S::COLS);
    const int kbs = (p.K + QK - 1) / QK;
    p.kb_chunk = (kbs + parts - 1) / parts;
    parts = (kbs + p.kb_chunk - 1) / p.kb_chunk;                 // no part without a block
    DEERS_SMEM_ONCE(ctx, (gemm_q8_split_kernel<I8, T, BN, SWAP>), S::SMEM);
    KernelTimerScope ts(ctx, DEERS_K_GEMM);
    DEERS_CUDA_TRY(ctx, launch_chained(ctx, gemm_q8_split_kernel<I8, T, BN, SWAP>, (unsigned)(tiles * parts), QS_THREADS, S::SMEM, parts, ta, tb, p));
    return DEERS_OK;
}

template <bool I8, typename T, bool PAIR>
int gemm_q8_whole(deers_ctx* ctx, const GemmQ8Params& p, const void* a, long long lda, const void* b, long long ldb, int room) {
    constexpr int BN = 256, TM = PAIR ? 2 * QM : QM, CTAS = PAIR ? 2 : 1;
    using S = QShape<BN, PAIR>;
    CUtensorMap ta, tb;
    int rc = tmap_bytes(ctx, &ta, a, p.M, p.K, lda, QM);
    if (!rc) rc = tmap_bytes(ctx, &tb, b, p.N, p.K, ldb, BN / CTAS);
    if (rc) return rc;
    const long long tiles = (long long)((p.M + TM - 1) / TM) * ((p.N + BN - 1) / BN);
    const unsigned grid = (unsigned)(tiles < room ? tiles : room);
    DEERS_SMEM_ONCE(ctx, (gemm_q8_kernel<I8, T, BN, PAIR>), S::SMEM);
    const ChainScope chain(ctx, tiles * ((p.K + QK - 1) / QK) / grid);
    KernelTimerScope ts(ctx, DEERS_K_GEMM);
    DEERS_CUDA_TRY(ctx, launch_chained(ctx, gemm_q8_kernel<I8, T, BN, PAIR>, grid * CTAS, Q_THREADS, S::SMEM, CTAS, ta, tb, p));
    return DEERS_OK;
}

template <bool I8, typename T>
int gemm_q8_launch(deers_ctx* ctx, const GemmQ8Params& p, const void* a, long long lda, const void* b, long long ldb) {
    int pairs;
    GemmQ8Plan plan;
    const int rc = plan_gemm_q8(ctx, p.M, p.N, p.K, &plan, &pairs);
    if (rc) return rc;
    if (plan.split) {
        const auto go = plan.swap ? (plan.bn == 16 ? gemm_q8_split<I8, T, 16, true> : plan.bn == 32 ? gemm_q8_split<I8, T, 32, true> : gemm_q8_split<I8, T, 64, true>)
                                  : (plan.bn == 128 ? gemm_q8_split<I8, T, 128, false> : gemm_q8_split<I8, T, 256, false>);
        return go(ctx, p, a, lda, b, ldb, plan.parts);
    }
    return plan.pair ? gemm_q8_whole<I8, T, true>(ctx, p, a, lda, b, ldb, pairs) : gemm_q8_whole<I8, T, false>(ctx, p, a, lda, b, ldb, ctx->sm_count);
}

}  // namespace

int route_gemm_q8(deers_ctx* ctx, int M, int N, int K, deers_product_route* r) {
    int pairs;
    GemmQ8Plan p;
    const int rc = plan_gemm_q8(ctx, M, N, K, &p, &pairs);
    if (rc) return rc;
    r->tile_m = p.swap ? p.bn : p.pair ? 2 * QM : QM; r->tile_n = p.swap ? QM : p.bn; r->parts = p.parts;
    r->tensor_core = 1; r->pair = p.pair; r->swapped = p.swap; r->persistent = !p.split;
    return DEERS_OK;
}

extern "C" int deers_b200_gemm_q8(deers_ctx* ctx, int32_t M, int32_t N, int32_t K, int32_t code, const void* a, int64_t lda, const float* a_scale,
                                  const void* b, int64_t ldb, const float* b_scale, int32_t out_dtype, void* c, int64_t ldc) {
    if (!ctx) return DEERS_ERR_NULL;
    if (code != DEERS_I8 && code != DEERS_E4M3) return DEERS_ERR_DTYPE;
    if (out_dtype != DEERS_F16 && out_dtype != DEERS_F32) return DEERS_ERR_DTYPE;
    if (M < 0 || N < 1 || K < 1) return DEERS_ERR_SHAPE;
    constexpr int MOST = 0x7fffffff - 512;                       // places behind the last row or column of a tile stay within 31 bits
    if (M > MOST || N > MOST || K > MOST) return DEERS_ERR_UNSUPPORTED;
    if (code == DEERS_I8 && K >= 131072) return DEERS_ERR_UNSUPPORTED;       // 2^31 / 128^2: sums stay whole numbers of 32 bits
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
