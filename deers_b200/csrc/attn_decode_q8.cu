// Decode-time attention over a cache of e4m3 codes with a scale for every 32 tokens of a head (cache_q8.cu writes it).
//
//     s_j = scale * ks[j / 32] * (q . k_j)      o = sum_j p_j vs[j / 32] v_j / sum_j p_j      p_j = exp(s_j - max)
//
// G query heads share a cached head, and each brings Tq new rows, so a cached key meets R = G * Tq query rows.  They are the eight columns
// (or twice eight) of mma.m16n8k16 products whose rows are keys: codes become f16 exactly, sums are f32.  With codes of one byte the kernel
// has half the time per value that an f16 cache leaves: by f32 instructions alone a value costs a conversion and a multiplication for
// every query row, by these products 0.5 to 0.75 conversion instructions and a 32nd of two products whatever R is up to eight.
//
//   A warp takes blocks of 32 keys (one scale each) in turn, which TMA brings into a ring of its own in shared memory (swizzled, so that lanes read
//   without conflicts, or two by two): a block costs one lane two copies, and warps wait for nobody but their own.
//   S^T = K Q^T: the order of the channels inside a product is free as long as K and Q agree, so a lane's 16 consecutive bytes of a key
//   are its share of four products.  O^T += V^T P^T: the order of the keys is free too, and a lane's bytes of two keys are interleaved by
//   byte permutations, which is the transposition that V needs.  P moves from the first product's layout to the second's by movmatrix.
//   Weights are exp(s - m) * vs / vref * 2^15 with running maxima m (per row) and vref, as two f16 each (22 bits): the block's scale of V
//   costs nothing per value, and small weights keep their bits.  q in f32 is two f16 as well, scaled per row by a power of two.
//   Warps meet in shared memory, the chunks of a slice in distributed shared memory (up to eight) or the workspace.
// A row that sees no key has o = 0 and lse = -inf.  What a row does not see does not reach it, not even a NaN stored there.
// Bound: HBM, one byte a value.
#include <cuda_fp16.h>

#include "common.cuh"
#include "q8_codes.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

#include <cooperative_groups.h>

int deers_check_cache(const deers_cache_q8* c);

namespace {

constexpr int DQ_WARPS = 4;
constexpr int DQ_MAX_SPLITS = 4 * 148;
constexpr float DQ_LOG2E = 1.4426950408889634f, DQ_LN2 = 0.6931471805599453f;
constexpr float DQ_UP = 32768.0f;                                // weights are at most 2^15 of f16's 65504

struct DecodeQ8Params {
    const void* q; void* o; float* lse;
    const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
    const int* lengths;
    float* part;                                                 // [slice][tile][split][rows of a tile][D + 2]
    long long sq[3], so[3], sk[3], sv[3], skl[2], svl[2];
    int H, G, Tq, D, cap, causal, splits, q_vec;
    float scale;
    unsigned int* err;
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// 2^x for x <= 0 (results below 2^-126 are zero).
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

// Shapes of a kernel for heads of up to DP channels and 8 * NT query rows.
template <int DP, int NT>
struct Shape {
    static constexpr int KC = DP / 64;                           // 16-byte pieces of a key that a lane owns: at 16 * (lane % 4 + 4 c)
    static constexpr int VB = DP >= 128 ? 16 : 8;                // bytes of a piece of V: at VB * (lane / 4 + 8 c)
    static constexpr int VC = DP / 8 / VB;
    static constexpr int STAGES = DP == 64 ? 4 : 2;
    static constexpr int STAGE_BYTES = 32 * 2 * DP;              // 32 keys, K and V
    static constexpr int BOX = DP == 64 ? 64 : 128, BOXES = DP / BOX;     // bytes of a key in a box of 32 keys, boxes of K or of V
    static constexpr int RING = DQ_WARPS * STAGES * STAGE_BYTES;
    static constexpr int ROWS = 8 * NT;
    static constexpr int OS = DP + 4;                            // row of partial results: O, then maximum and sum
    static constexpr int MERGE = DQ_WARPS * ROWS * OS * 4;
    static constexpr int PART = ROWS * OS * 4;
    static constexpr int BARS = RING > MERGE + PART ? RING : MERGE + PART;         // (the ring has been read when the warps meet)
    static constexpr int SMEM = BARS + DQ_WARPS * STAGES * 8 + 16;
};

enum DecodeQ8End { DQ_ONE_CHUNK = 0, DQ_CLUSTER = 1, DQ_TO_WORKSPACE = 2 };

// Barriers: nothing of global memory.
template <int DP, int NT>
__device__ __forceinline__ void decode_q8_prologue(const void* tmap_k, const void* tmap_v) {
    using S = Shape<DP, NT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BARS);
    uint32_t* abort_s = reinterpret_cast<uint32_t*>(bars + DQ_WARPS * S::STAGES);
    if (threadIdx.x == 0) {
        for (int i = 0; i < DQ_WARPS * S::STAGES; ++i) sm100::mbar_init(&bars[i], 1);
        abort_s[0] = 0;
        sm100::fence_barrier_init();
        sm100::tma_prefetch_desc(tmap_k); sm100::tma_prefetch_desc(tmap_v);
    }
}

template <typename T, int DP, int NT, int END>
__global__ void __launch_bounds__(32 * DQ_WARPS)
decode_q8_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const DecodeQ8Params p) {
    decode_q8_prologue<DP, NT>(&tmap_k, &tmap_v);
    chain_wait();
    using S = Shape<DP, NT>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int QP = F32 ? 2 : 1;                              // f16 parts of a value of q
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, Hkv = p.H / p.G, b = blockIdx.y / Hkv, kvh = blockIdx.y % Hkv, tile = blockIdx.z;
    const int R = p.G * p.Tq, row0 = tile * S::ROWS;
    int len = p.lengths[b];
    if (len < 0 || len > p.cap) {
        if (threadIdx.x == 0) atomicCAS(p.err, 0u, (unsigned)DEERS_KERR_CACHE | 2u);
        len = min(max(len, 0), p.cap);
    }
    // this block's keys: its share of the sequence's blocks of 32
    const int blocks = (len + 31) / 32;
    const int blk0 = (int)((long long)blocks * split / p.splits), blk1 = (int)((long long)blocks * (split + 1) / p.splits);
    const uint8_t* vb = p.v + b * p.sv[0] + kvh * p.sv[1];
    const float* ksl = p.k_scale + b * p.skl[0] + kvh * p.skl[1];
    const float* vsl = p.v_scale + b * p.svl[0] + kvh * p.svl[1];

    __syncthreads();                                             // the barriers are there
    uint8_t* ring = smem + warp * (S::STAGES * S::STAGE_BYTES);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::BARS) + warp * S::STAGES;
    const sm100::WaitState ws{reinterpret_cast<uint32_t*>(smem + S::BARS + DQ_WARPS * S::STAGES * 8), p.err};
    // Block `blk` into stage s, by one lane.  (Keys behind the sequence's last may lie in it, and are masked below.)
    auto fetch = [&](int blk, int s) {
        if (blk < blk1 && lane == 0) {
            sm100::mbar_arrive_expect_tx(&full[s], S::STAGE_BYTES);
#pragma unroll
            for (int i = 0; i < S::BOXES; ++i) {
                sm100::tma_load_4d(ring + s * S::STAGE_BYTES + i * 32 * S::BOX, &tmap_k, &full[s], i * S::BOX, blk * 32, kvh, b);
                sm100::tma_load_4d(ring + s * S::STAGE_BYTES + 32 * DP + i * 32 * S::BOX, &tmap_v, &full[s], i * S::BOX, blk * 32, kvh, b);
            }
        }
    };
    // 16 bytes of key j at 16 * piece (bytes 8 * half of them) inside the boxes of K or of V
    auto in_boxes = [&](int j, int piece) {
        if constexpr (DP == 64) return j * 64 + ((piece ^ (j >> 1 & 3)) << 4);
        else return (piece >> 3) * (32 * 128) + j * 128 + (((piece & 7) ^ (j & 7)) << 4);
    };
    // This lane's keys of a block: 8 r + g of K; 2t, 2t + 1, 2t + 8, 2t + 9 of either half of V.
    const auto v_key = [&](int r) { return (r >> 2) * 16 + ((r >> 1) & 1) * 8 + 2 * t + (r & 1); };
    const auto v_at = [&](int r, int c) { return 32 * DP + (DP == 64 ? in_boxes(v_key(r), g >> 1) + 8 * (g & 1) : in_boxes(v_key(r), g + 8 * c)); };
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; ++s) fetch(blk0 + warp + s * DQ_WARPS, s);

    // q as the products' second operand: lane (g, t) has row g, channels 16 (t + 4 c) ..
    uint32_t qf[NT][QP][S::KC][8];
    float qs[NT][2];                                             // factor of the scores of rows 2t, 2t + 1
    int lim[NT][2];                                              // keys that they see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + nt * 8 + g;
        float f[S::KC][16];
        const T* src = static_cast<const T*>(p.q);
        if (r < R) src += b * p.sq[0] + (long long)(kvh * p.G + r / p.Tq) * p.sq[1] + (long long)(r % p.Tq) * p.sq[2];
#pragma unroll
        for (int c = 0; c < S::KC; ++c) {
            const int d = 16 * (t + 4 * c);
            if (r < R && d < p.D) {
                if (p.q_vec) {
                    T raw[16];
#pragma unroll
                    for (int w = 0; w < (int)sizeof(T); ++w) reinterpret_cast<uint4*>(raw)[w] = reinterpret_cast<const uint4*>(src + d)[w];
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[c][e] = (float)raw[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[c][e] = (float)src[d + e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) f[c][e] = 0.f;
            }
        }
        float back = 1.f;
        if constexpr (F32) {
            unsigned top = 0;
#pragma unroll
            for (int c = 0; c < S::KC; ++c)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(f[c][e]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // a power of two that brings the largest value to 2^14 .. 2^15 (exponents of factor and inverse both in range)
            int e = 141 - (int)(top >> 23);
            e = top == 0 || top >= 0x7f800000u ? 0 : max(-100, min(100, e));
            const float up = __uint_as_float((unsigned)(127 + e) << 23);
            back = __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
            for (int c = 0; c < S::KC; ++c)
#pragma unroll
                for (int k = 0; k < 16; ++k) f[c][k] *= up;
        }
#pragma unroll
        for (int c = 0; c < S::KC; ++c)
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                qf[nt][0][c][w] = pack2(f[c][2 * w], f[c][2 * w + 1]);
                if constexpr (F32) {
                    const float2 hi = unpack2(qf[nt][0][c][w]);
                    qf[nt][1][c][w] = pack2(f[c][2 * w] - hi.x, f[c][2 * w + 1] - hi.y);
                }
            }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int rx = row0 + nt * 8 + 2 * t + x;
            qs[nt][x] = __shfl_sync(0xffffffffu, back, (2 * t + x) * 4) * p.scale * DQ_LOG2E;
            lim[nt][x] = p.causal && rx < R ? len - (p.Tq - 1 - rx % p.Tq) : len;      // (rows that are not: zeros, never written)
        }
    }
    const int lim_min = p.causal ? len - (p.Tq - 1) : len;       // keys that every row sees

    float o[NT][DP / 16][4], m[NT][2], l[NT][2], vref = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
    }

    int stage = 0;
    uint32_t phase = 0;
    float ks_next = 0.f, vs_next = 0.f;                          // scales of the next round's block
    if (blk0 + warp < blk1) { ks_next = ksl[blk0 + warp]; vs_next = vsl[blk0 + warp]; }
#pragma unroll 1
    for (int blk = blk0 + warp; blk < blk1; blk += DQ_WARPS) {
        const float ks = ks_next, vs = vs_next;
        if (blk + DQ_WARPS < blk1) { ks_next = ksl[blk + DQ_WARPS]; vs_next = vsl[blk + DQ_WARPS]; }
        __syncwarp();
        fetch(blk + (S::STAGES - 1) * DQ_WARPS, stage == 0 ? S::STAGES - 1 : stage - 1);      // (the stage that the last round has read)
        if (!sm100::mbar_wait_warp(ws, &full[stage], phase, DEERS_KERR_CACHE | 3u)) break;
        const uint8_t* st = ring + stage * S::STAGE_BYTES;
        // ---- scores: keys 16 mt + g and 16 mt + g + 8.  The tensor core cuts its sums off, towards zero: with f32 queries the chains are short (a
        // piece of a key each, the low parts of q apart) and added in f32.
        float s[NT][2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            constexpr int CHAINS = F32 ? S::KC + 1 : 1;
            float sum[NT][CHAINS][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < CHAINS; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[nt][i][e] = 0.f;
#pragma unroll
            for (int c = 0; c < S::KC; ++c) {
                const uint4 x = *reinterpret_cast<const uint4*>(st + in_boxes(16 * mt + g, t + 4 * c));
                const uint4 y = *reinterpret_cast<const uint4*>(st + in_boxes(16 * mt + 8 + g, t + 4 * c));
                const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t a0 = q8::e4m3_lo(xw[w]), a2 = q8::e4m3_hi(xw[w]), a1 = q8::e4m3_lo(yw[w]), a3 = q8::e4m3_hi(yw[w]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816(sum[nt][F32 ? c : 0], a0, a1, a2, a3, qf[nt][0][c][2 * w], qf[nt][0][c][2 * w + 1]);
                        if constexpr (F32) mma16816(sum[nt][S::KC], a0, a1, a2, a3, qf[nt][1][c][2 * w], qf[nt][1][c][2 * w + 1]);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float z = sum[nt][CHAINS - 1][e];
#pragma unroll
                    for (int i = 0; i < CHAINS - 1; ++i) z += sum[nt][i][e];
                    s[nt][mt][e] = z;
                }
        }
        // ---- running maxima
        const bool edge = blk * 32 + 32 > lim_min;               // (uniform)
        const float vnew = fmaxf(vref, vs), vfac = vnew > 0.f ? vref / vnew : 0.f, vw = vnew > 0.f ? vs / vnew * DQ_UP : 0.f;
        bool moved = vnew != vref;
        vref = vnew;
        float fac[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float f = qs[nt][x] * ks;
                float mx = m[nt][x];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int y = 0; y < 2; ++y) s[nt][mt][2 * y + x] *= f;
                if (edge) {
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                        for (int y = 0; y < 2; ++y)
                            if (blk * 32 + mt * 16 + y * 8 + g >= lim[nt][x]) s[nt][mt][2 * y + x] = -INFINITY;
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int y = 0; y < 2; ++y) mx = fmaxf(mx, s[nt][mt][2 * y + x]);
#pragma unroll
                for (int off = 4; off <= 16; off *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                // (-inf: nothing seen so far, or NaN alone, which have to reach the sums)
                const float ms = mx == -INFINITY ? 0.f : mx;
                fac[nt][x] = power2(m[nt][x] - ms);
                moved |= mx != m[nt][x];
                m[nt][x] = mx;
                l[nt][x] *= fac[nt][x];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float pj = power2(s[nt][mt][2 * y + x] - ms);
                        l[nt][x] += pj;
                        s[nt][mt][2 * y + x] = pj;
                    }
            }
        if (!F32 && __any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < DP / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][j][e] *= fac[nt][e & 1] * vfac;
        }
        // ---- weights, transposed
        uint32_t pw[NT][2][2][2];                                // [tile][16 keys][part][8 keys]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float w0 = s[nt][mt][2 * y] * vw, w1 = s[nt][mt][2 * y + 1] * vw;
                    const uint32_t hi = pack2(w0, w1);
                    const float2 h = unpack2(hi);
                    pw[nt][mt][0][y] = transposed(hi);
                    pw[nt][mt][1][y] = transposed(pack2(w0 - h.x, w1 - h.y));
                }
        // A weight of zero does not keep out a NaN: where a key that some rows do not see holds one, the rows' sums are made one by one.
        if (edge && lim_min < len) {
            uint32_t nan = 0;
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int c = 0; c < S::VC; ++c) {
                    if (v_key(r) >= len - blk * 32) continue;
#pragma unroll
                    for (int w = 0; w < S::VB / 4; ++w)
                        nan |= ((reinterpret_cast<const uint32_t*>(st + v_at(r, c))[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                }
            if (__any_sync(0xffffffffu, nan != 0)) {
                if constexpr (F32) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nt][j][e] *= fac[nt][e & 1] * vfac;
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll 1
                        for (int i = 0; i < 8; ++i) {
                            const int key = blk * 32 + mt * 16 + y * 8 + i;
                            const uint8_t* row = vb + (long long)min(key, len - 1) * p.sv[2];
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float w[2];
#pragma unroll
                                for (int x = 0; x < 2; ++x) w[x] = __shfl_sync(0xffffffffu, s[nt][mt][2 * y + x], i * 4 + t) * vw;
#pragma unroll
                                for (int j = 0; j < DP / 16; ++j) {
                                    const int d = S::VB * (g + 8 * (j / (S::VB / 2))) + 2 * (j % (S::VB / 2));
                                    float f[4];
                                    q8::e4m3_values(d < p.D ? *reinterpret_cast<const uint16_t*>(row + d) : 0u, f);
#pragma unroll
                                    for (int e = 0; e < 4; ++e)
                                        if (key < lim[nt][e & 1]) o[nt][j][e] = fmaf(w[e & 1], f[e >> 1], o[nt][j][e]);
                                }
                            }
                        }
                if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
                continue;
            }
        }
        // ---- values.  With f32 queries a block's sums start from zero and are added to O, scaled anew on the way, in f32.
#pragma unroll
        for (int c = 0; c < S::VC; ++c) {
            constexpr int VW = S::VB / 4;
            uint32_t x[2][4][VW];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint8_t* src = st + v_at(4 * mt + r, c);
                    if constexpr (VW == 4) *reinterpret_cast<uint4*>(x[mt][r]) = *reinterpret_cast<const uint4*>(src);
                    else *reinterpret_cast<uint2*>(x[mt][r]) = *reinterpret_cast<const uint2*>(src);
                }
            if (blk * 32 + 32 > len) {                           // what lies behind the last key is nobody's, and may be NaN
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (v_key(4 * mt + r) >= len - blk * 32) {
#pragma unroll
                            for (int w = 0; w < VW; ++w) x[mt][r][w] = 0;
                        }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int j = c * (S::VB / 2) + 2 * w + k;               // channels VB (g + 8 c) + 4 w + 2 k and the next
                    uint32_t a[2][4];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const uint32_t e0 = __byte_perm(x[mt][0][w], x[mt][1][w], k ? 0x7362 : 0x5140), e1 = __byte_perm(x[mt][2][w], x[mt][3][w], k ? 0x7362 : 0x5140);
                        a[mt][0] = q8::e4m3_lo(e0); a[mt][1] = q8::e4m3_hi(e0); a[mt][2] = q8::e4m3_lo(e1); a[mt][3] = q8::e4m3_hi(e1);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if constexpr (F32) {
                            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int part = 1; part >= 0; --part)
#pragma unroll
                                for (int mt = 0; mt < 2; ++mt) mma16816(sum, a[mt][0], a[mt][1], a[mt][2], a[mt][3], pw[nt][mt][part][0], pw[nt][mt][part][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nt][j][e] = fmaf(o[nt][j][e], fac[nt][e & 1] * vfac, sum[e]);
                        } else {
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                                for (int part = 0; part < 2; ++part) mma16816(o[nt][j], a[mt][0], a[mt][1], a[mt][2], a[mt][3], pw[nt][mt][part][0], pw[nt][mt][part][1]);
                        }
                    }
                }
        }
        if (++stage == S::STAGES) { stage = 0; phase ^= 1u; }
    }
    chain_next();

    // ---- the warps meet
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int off = 4; off <= 16; off *= 2) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], off);
    __syncthreads();                                             // every ring has been read
    float* meet = reinterpret_cast<float*>(smem);
    float* part = reinterpret_cast<float*>(smem + S::MERGE);
    {
        float* mine = meet + warp * S::ROWS * S::OS;
        const float down = vref * (1.0f / DQ_UP);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                const int d = S::VB * (g + 8 * (j / (S::VB / 2))) + 2 * (j % (S::VB / 2));
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[(nt * 8 + 2 * t + (e & 1)) * S::OS + d + (e >> 1)] = o[nt][j][e] * down;
            }
            if (g == 0) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mine[(nt * 8 + 2 * t + x) * S::OS + DP] = m[nt][x];
                    mine[(nt * 8 + 2 * t + x) * S::OS + DP + 1] = l[nt][x];
                }
            }
        }
    }
    __syncthreads();
    const int rows = min(S::ROWS, R - row0);
    auto out_row = [&](int r) {
        const int rr = row0 + r;
        return static_cast<T*>(p.o) + b * p.so[0] + (long long)(kvh * p.G + rr / p.Tq) * p.so[1] + (long long)(rr % p.Tq) * p.so[2];
    };
    auto lse_at = [&](int r) {
        const int rr = row0 + r;
        return p.lse + ((long long)b * p.H + kvh * p.G + rr / p.Tq) * p.Tq + rr % p.Tq;
    };
    // n partial rows at `from`, `step` floats apart: (maximum, sum, O) of the whole
    auto joined = [&](const float* from, int step, int r, int d, float& mx, float& sum) {
        mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < DQ_WARPS; ++w) mx = fmaxf(mx, from[w * step + r * S::OS + DP]);
        const float ms = mx == -INFINITY ? 0.f : mx;
        float v = 0.f;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < DQ_WARPS; ++w) {
            const float* at = from + w * step + r * S::OS;
            const float f = exp2f(at[DP] - ms);
            sum = fmaf(f, at[DP + 1], sum);
            v = fmaf(f, at[d], v);
        }
        return v;
    };
    float* to_part = END == DQ_TO_WORKSPACE ? p.part + (((long long)blockIdx.y * gridDim.z + tile) * p.splits + split) * (S::ROWS * (p.D + 2)) : nullptr;
    for (int i = threadIdx.x; i < rows * p.D; i += 32 * DQ_WARPS) {
        const int r = i / p.D, d = i % p.D;
        float mx, sum;
        const float v = joined(meet, S::ROWS * S::OS, r, d, mx, sum);
        if constexpr (END == DQ_ONE_CHUNK) {
            put(out_row(r) + d, sum == 0.f ? 0.f : v / sum);
            if (p.lse && d == 0) *lse_at(r) = (mx + log2f(sum)) * DQ_LN2;
        } else if constexpr (END == DQ_CLUSTER) {
            part[r * S::OS + d] = v;
            if (d == 0) { part[r * S::OS + DP] = mx; part[r * S::OS + DP + 1] = sum; }
        } else {
            to_part[r * (p.D + 2) + d] = v;
            if (d == 0) { to_part[r * (p.D + 2) + p.D] = mx; to_part[r * (p.D + 2) + p.D + 1] = sum; }
        }
    }
    if constexpr (END == DQ_CLUSTER) {
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster.sync();
        const float* from[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) from[z] = cluster.map_shared_rank(part, z < p.splits ? z : 0);
        for (int i = split * 32 * DQ_WARPS + threadIdx.x; i < rows * p.D; i += p.splits * 32 * DQ_WARPS) {
            const int r = i / p.D, d = i % p.D;
            float w[8], mx = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                w[z] = z < p.splits ? from[z][r * S::OS + DP] : -INFINITY;
                mx = fmaxf(mx, w[z]);
            }
            const float ms = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int z = 0; z < 8; ++z)
                if (z < p.splits) {
                    const float f = exp2f(w[z] - ms);
                    sum = fmaf(f, from[z][r * S::OS + DP + 1], sum);
                    v = fmaf(f, from[z][r * S::OS + d], v);
                }
            put(out_row(r) + d, sum == 0.f ? 0.f : v / sum);
            if (p.lse && d == 0) *lse_at(r) = (mx + log2f(sum)) * DQ_LN2;
        }
        cluster.sync();                                          // nobody leaves while a peer still reads its part
    }
}

// Joins the chunks of a slice's rows from the workspace: a block per (row of a tile, tile, slice).
template <typename T>
__global__ void __launch_bounds__(128) decode_q8_join_kernel(const DecodeQ8Params p, int tile_rows, int tiles) {
    chain_begin();
    __shared__ float s_w[DQ_MAX_SPLITS], s_r[8];
    const int r = blockIdx.x, tile = blockIdx.z, Hkv = p.H / p.G, b = blockIdx.y / Hkv, kvh = blockIdx.y % Hkv;
    const int rr = tile * tile_rows + r, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (rr >= p.G * p.Tq) return;
    const long long step = (long long)tile_rows * (p.D + 2);
    const float* part = p.part + ((long long)blockIdx.y * tiles + tile) * p.splits * step + r * (p.D + 2);
    float mx = -INFINITY;
    for (int z = threadIdx.x; z < p.splits; z += 128) {
        s_w[z] = part[z * step + p.D];
        mx = fmaxf(mx, s_w[z]);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    if (lane == 0) s_r[warp] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(s_r[0], s_r[1]), fmaxf(s_r[2], s_r[3]));
    const float ms = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    for (int z = threadIdx.x; z < p.splits; z += 128) {
        const float w = exp2f(s_w[z] - ms);
        s_w[z] = w;
        sum = fmaf(w, part[z * step + p.D + 1], sum);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) s_r[4 + warp] = sum;
    __syncthreads();
    sum = (s_r[4] + s_r[5]) + (s_r[6] + s_r[7]);
    const int head = kvh * p.G + rr / p.Tq, i = rr % p.Tq;
    T* o = static_cast<T*>(p.o) + b * p.so[0] + head * p.so[1] + i * p.so[2];
    for (int d = threadIdx.x; d < p.D; d += 128) {
        float v = 0.f;
        for (int z = 0; z < p.splits; ++z) v = fmaf(s_w[z], part[z * step + d], v);
        put(o + d, sum == 0.f ? 0.f : v / sum);
    }
    if (p.lse && threadIdx.x == 0) p.lse[((long long)b * p.H + head) * p.Tq + i] = (mx + log2f(sum)) * DQ_LN2;
}

struct DecodeQ8Plan { int dp, nt, tiles, splits, end; };

// How the work is cut.  Sixteen query rows share a walk where there are more than eight (heads up to 128 wide: the registers hold their O).
// The slices' keys are cut so that every SM has two blocks: up to eight chunks meet as a cluster, more through the workspace.
DecodeQ8Plan plan_decode_q8(const deers_decode_q8_desc* d) {
    DecodeQ8Plan p;
    p.dp = d->cache.D <= 64 ? 64 : d->cache.D <= 128 ? 128 : 256;
    const int R = d->H / d->cache.H * d->Tq;
    p.nt = R > 8 && p.dp <= 128 ? 2 : 1;
    p.tiles = (R + 8 * p.nt - 1) / (8 * p.nt);
    const long long slices = (long long)d->cache.B * d->cache.H * p.tiles;
    const long long blocks = (d->cache.capacity + 31) / 32;
    long long want = (2 * 148 + slices - 1) / slices;
    const long long most = (blocks + 7) / 8;                     // at least 256 keys a chunk
    if (want > most) want = most;
    if (want > DQ_MAX_SPLITS) want = DQ_MAX_SPLITS;
    if (want < 1) want = 1;
    p.splits = (int)want;
    p.end = want == 1 ? DQ_ONE_CHUNK : want <= 8 ? DQ_CLUSTER : DQ_TO_WORKSPACE;
    return p;
}

size_t decode_q8_bytes(const deers_decode_q8_desc* d, const DecodeQ8Plan& p) {
    if (p.end != DQ_TO_WORKSPACE) return 0;
    return (size_t)d->cache.B * d->cache.H * p.tiles * p.splits * (8 * p.nt) * (d->cache.D + 2) * sizeof(float);
}

int decode_q8_check(const deers_decode_q8_desc* d) {
    if (!d) return DEERS_ERR_NULL;
    if (d->dtype != DEERS_F16 && d->dtype != DEERS_F32) return DEERS_ERR_DTYPE;
    const int rc = deers_check_cache(&d->cache);
    if (rc) return rc;
    if (d->H < 1 || d->Tq < 1 || d->H % d->cache.H) return DEERS_ERR_SHAPE;
    if (!(d->scale == d->scale)) return DEERS_ERR_SHAPE;
    if (d->Tq > 128 || d->Tq > d->cache.capacity || (long long)d->cache.B * d->cache.H > 65535 || (long long)d->H / d->cache.H * d->Tq > 65535)
        return DEERS_ERR_UNSUPPORTED;
    // (maps of the copies want strides that advance)
    if (d->cache.B > 1 && (d->cache.k_strides[0] == 0 || d->cache.v_strides[0] == 0)) return DEERS_ERR_LAYOUT;
    if (d->cache.H > 1 && (d->cache.k_strides[1] == 0 || d->cache.v_strides[1] == 0)) return DEERS_ERR_LAYOUT;
    for (const int64_t* s : {d->q_strides, d->o_strides}) {
        if (s[3] != 1) return DEERS_ERR_LAYOUT;
        for (int i = 0; i < 3; ++i)
            if (s[i] < 0) return DEERS_ERR_LAYOUT;
    }
    return DEERS_OK;
}

// Map over the codes of a cache, [D, capacity, H, B] (innermost first): boxes of 32 keys, zeros outside.
int tmap_cache(deers_ctx* ctx, CUtensorMap* out, const void* base, const deers_cache_q8& c, const int64_t* st, int box) {
    const cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.capacity, (cuuint64_t)c.H, (cuuint64_t)c.B};
    // (an axis of one place never advances: any legal stride)
    const cuuint64_t t = (cuuint64_t)st[2], h = c.H > 1 ? (cuuint64_t)st[1] : t * dims[1], b = c.B > 1 ? (cuuint64_t)st[0] : h * dims[2];
    const cuuint64_t strides[3] = {t, h, b};
    const cuuint32_t boxes[4] = {(cuuint32_t)box, 32, 1, 1};
    return make_tmap_bytes(ctx, out, base, dims, strides, boxes, box == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int DP, int NT>
int decode_q8_launch(deers_ctx* ctx, const DecodeQ8Params& p, const DecodeQ8Plan& plan, int slices, const deers_cache_q8& cache) {
    using S = Shape<DP, NT>;
    CUtensorMap tk, tv;
    int rc = tmap_cache(ctx, &tk, cache.k, cache, cache.k_strides, S::BOX);
    if (!rc) rc = tmap_cache(ctx, &tv, cache.v, cache, cache.v_strides, S::BOX);
    if (rc) return rc;
    const dim3 grid(plan.splits, slices, plan.tiles);
    if (plan.end == DQ_ONE_CHUNK) {
        DEERS_SMEM_ONCE(ctx, (decode_q8_kernel<T, DP, NT, DQ_ONE_CHUNK>), S::SMEM);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_kernel<T, DP, NT, DQ_ONE_CHUNK>, grid, 32 * DQ_WARPS, S::SMEM, 1, tk, tv, p));
    } else if (plan.end == DQ_CLUSTER) {
        DEERS_SMEM_ONCE(ctx, (decode_q8_kernel<T, DP, NT, DQ_CLUSTER>), S::SMEM);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_kernel<T, DP, NT, DQ_CLUSTER>, grid, 32 * DQ_WARPS, S::SMEM, plan.splits, tk, tv, p));
    } else {
        DEERS_SMEM_ONCE(ctx, (decode_q8_kernel<T, DP, NT, DQ_TO_WORKSPACE>), S::SMEM);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_kernel<T, DP, NT, DQ_TO_WORKSPACE>, grid, 32 * DQ_WARPS, S::SMEM, 1, tk, tv, p));
        const dim3 rows(S::ROWS, slices, plan.tiles);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_join_kernel<T>, rows, 128, 0, 1, p, S::ROWS, plan.tiles));
        ctx->launches += 1;
    }
    return DEERS_OK;
}

template <typename T>
int decode_q8_widths(deers_ctx* ctx, const DecodeQ8Params& p, const DecodeQ8Plan& plan, int slices, const deers_cache_q8& c) {
    if (plan.dp == 64) return plan.nt == 2 ? decode_q8_launch<T, 64, 2>(ctx, p, plan, slices, c) : decode_q8_launch<T, 64, 1>(ctx, p, plan, slices, c);
    if (plan.dp == 128) return plan.nt == 2 ? decode_q8_launch<T, 128, 2>(ctx, p, plan, slices, c) : decode_q8_launch<T, 128, 1>(ctx, p, plan, slices, c);
    return decode_q8_launch<T, 256, 1>(ctx, p, plan, slices, c);
}

}  // namespace

extern "C" size_t deers_b200_attn_decode_q8_workspace_bytes(const deers_decode_q8_desc* d) {
    return decode_q8_check(d) == DEERS_OK ? decode_q8_bytes(d, plan_decode_q8(d)) : 0;
}

extern "C" int deers_b200_attn_decode_q8(deers_ctx* ctx, const deers_decode_q8_desc* d, const void* q, const int32_t* lengths, void* o, float* lse,
                                         void* workspace, size_t workspace_bytes) {
    if (!ctx || !d) return DEERS_ERR_NULL;
    int rc = decode_q8_check(d);
    if (rc) return rc;
    if (!q || !lengths || !o) return DEERS_ERR_NULL;
    const uintptr_t es = d->dtype == DEERS_F16 ? 2 : 4;
    if (((uintptr_t)q | (uintptr_t)o) & (es - 1) || ((uintptr_t)lengths | (uintptr_t)lse) & 3u) return DEERS_ERR_LAYOUT;
    const DecodeQ8Plan plan = plan_decode_q8(d);
    const size_t need = decode_q8_bytes(d, plan);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 3u))) return DEERS_ERR_WORKSPACE;
    DEERS_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    const deers_cache_q8& c = d->cache;
    DecodeQ8Params p;
    p.q = q; p.o = o; p.lse = lse; p.lengths = lengths; p.part = (float*)workspace;
    p.k = (const uint8_t*)c.k; p.v = (const uint8_t*)c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
    for (int i = 0; i < 3; ++i) { p.sq[i] = d->q_strides[i]; p.so[i] = d->o_strides[i]; p.sk[i] = c.k_strides[i]; p.sv[i] = c.v_strides[i]; }
    for (int i = 0; i < 2; ++i) { p.skl[i] = c.k_scale_strides[i]; p.svl[i] = c.v_scale_strides[i]; }
    p.H = d->H; p.G = d->H / c.H; p.Tq = d->Tq; p.D = c.D; p.cap = c.capacity; p.causal = d->causal; p.splits = plan.splits;
    p.scale = d->scale; p.err = ctx->dev_err;
    const int64_t al = 16 / (int64_t)es - 1;
    p.q_vec = ((uintptr_t)q & 15u) == 0 && ((d->q_strides[0] | d->q_strides[1] | d->q_strides[2]) & al) == 0;
    {
        KernelTimerScope ts(ctx, DEERS_K_DECODE);
        rc = d->dtype == DEERS_F16 ? decode_q8_widths<__half>(ctx, p, plan, c.B * c.H, c) : decode_q8_widths<float>(ctx, p, plan, c.B * c.H, c);
        if (rc) return rc;
    }
    ctx->launches += 1;
    DEERS_CUDA_TRY(ctx, cudaGetLastError());
    return DEERS_OK;
}
