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
//   Weights are exp(s - m) * vs * 2^K with a running maximum m, as two f16 each (22 bits): the block's scale of V costs nothing per value.  The power of two
//   is each row's own and follows the largest exp(s - m) * vs so far, to bring it to 2^14 .. 2^15: it is products of weight and scale that keep their
//   bits, whatever lies in blocks that a row gives no weight.  q in f32 is two f16 as well, scaled per row by a power of two.
//   Warps meet in shared memory, the chunks of a slice in distributed shared memory (up to eight) or the workspace.
// A row that sees no key has o = 0 and lse = -inf.  What a row does not see does not reach it, not even a NaN stored there.
// Bound: HBM, one byte a value, where slices fill the device evenly (64 x 32 heads of 2048 keys of 128, f16 161 us, 1.03 of the copy rate); with f32 queries and sixteen
// rows instructions (two f16 parts of q and of the weights: 3 x 4 heads of 20000 to 65000 keys of 96 36 to 39 us of 15); with ragged lengths the blocks
// that get the longest (see plan_decode_q8).
#include <cuda_fp16.h>

#include "common.cuh"
#include "q8_codes.cuh"
#include "sm100_ptx.cuh"
#include "tma_host.cuh"

#include <cooperative_groups.h>

int deers_check_cache(const deers_cache_q8* c);

namespace {

constexpr int DQ_WARPS = 4;
constexpr int DQ_MAX_SHARES = 2 * 148, DQ_MAX_EVEN = 64;         // even shares: blocks of threads and slices at most
constexpr int DQ_LONG = 16384;                                   // keys of a long slice
constexpr float DQ_LOG2E = 1.4426950408889634f, DQ_LN2 = 0.6931471805599453f;
constexpr int DQ_UP = 15;                                        // weights are at most 2^15 of f16's 65504

struct DecodeQ8Params {
    const void* q; void* o; float* lse;
    const uint8_t* k; const uint8_t* v; const float* k_scale; const float* v_scale;
    const int* lengths;
    float* part;                                                 // DQ_EVEN: [block of threads][rows of a tile][D + 4]: O, maximum, sum
    long long sq[3], so[3], sk[3], sv[3], skl[2], svl[2];
    int B, H, G, Tq, D, cap, causal, splits, tiles, q_vec, o_vec;
    float scale;
    unsigned int* err;
    unsigned int* told;                                          // of lengths outside of the cache
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

// 2^e, e in [-126, 127].
__device__ __forceinline__ float power2_of(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }

__device__ __forceinline__ void add4(float4& v, float w, const float4& x) {
    v.x = fmaf(w, x.x, v.x); v.y = fmaf(w, x.y, v.y); v.z = fmaf(w, x.z, v.z); v.w = fmaf(w, x.w, v.w);
}
__device__ __forceinline__ void send4(uint32_t to, const float4& v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void send(uint32_t to, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory"); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
// Four channels; vec: rows of o lie on 16-byte boundaries.
__device__ __forceinline__ void put4(float* p, const float4& v, int vec) {
    if (vec) *reinterpret_cast<float4*>(p) = v;
    else { p[0] = v.x; p[1] = v.y; p[2] = v.z; p[3] = v.w; }
}
__device__ __forceinline__ void put4(__half* p, const float4& v, int vec) {
    if (vec) *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    else { put(p, v.x); put(p + 1, v.y); put(p + 2, v.z); put(p + 3, v.w); }
}

// Shapes of a kernel for heads of up to DP channels (32, 64, 96, 128 or 256) and 8 * NT query rows.
//   K: a lane (g, t) has the channels 16 (t + 4 c) .. + 15 of a key, c < KC, and of DP = 32 or 96 the last 32's 8 t .. + 7: four to a product step
//   V: the channels VB (g + 8 c) .. + VB - 1, c < VC, and the last 32's 4 g .. + 3: two to a product tile
template <int DP, int NT>
struct Shape {
    static constexpr bool TAIL = DP % 64 != 0;
    static constexpr int KC = DP / 64, KS = DP / 16;             // 16-byte pieces; steps
    static constexpr int VB = DP % 128 == 0 ? 16 : 8, VC = (DP - 32 * TAIL) / 8 / VB, VT = DP / 16;      // bytes of a piece, pieces; tiles
    static constexpr int BOX = DP <= 64 ? 64 : 128, BOXES = DP == 256 ? 2 : 1;       // bytes of a key in a box of 32 keys (zeros behind D), boxes of K or of V
    static constexpr int HALF_STAGE = 32 * BOX * BOXES, STAGE_BYTES = 2 * HALF_STAGE;         // K, V
    static constexpr int STAGES = DP <= 64 ? 4 : 2;
    static constexpr int RING = DQ_WARPS * STAGES * STAGE_BYTES;
    static constexpr int ROWS = 8 * NT;
    static constexpr int OS = DP + 4;                            // row of partial results: O, then maximum and sum
    static constexpr int MERGE = DQ_WARPS * ROWS * OS * 4;
    static constexpr int PART = ROWS * DP * 4;                   // DQ_CLUSTER: [block][its share of O] and, before, [block][row] maximum and sum
    // (the ring has been read when the warps meet; what other blocks of a cluster send has a place of its own)
    static constexpr int SENT = RING > MERGE ? RING : MERGE, BARS = SENT + 8 * ROWS * 8 + PART + 8 * 32;
    static constexpr int SMEM = BARS + DQ_WARPS * STAGES * 8 + 16;
    // Blocks of threads on an SM: what shared memory has place for, or two where sixteen rows' registers count (with q in shared memory instead three
    // go on, and are slower: 39 -> 44 us for 37 x 8 slices of 2048 keys of 128, G 16, f16).
    static constexpr int ON_AN_SM = DP == 256 ? 1 : NT == 2 && DP >= 96 ? 2 : 3;
    // first of the four channels of product step i, of the two channels of tile j (a tile's rows 8 to 15 are the next ones)
    static __device__ __forceinline__ int k_channel(int i, int t) { return i < 4 * KC ? 16 * (t + 4 * (i / 4)) + 4 * (i % 4) : DP - 32 + 8 * t + 4 * (i - 4 * KC); }
    static __device__ __forceinline__ int v_channel(int j, int g) {
        return j < VC * (VB / 2) ? VB * (g + 8 * (j / (VB / 2))) + 2 * (j % (VB / 2)) : DP - 32 + 4 * g + 2 * (j - VC * (VB / 2));
    }
};

// What a block of threads works on: the keys of a slice (a head's rows of a tile of query rows), a share of them as one of a cluster, or an even share of
// all blocks of all slices, whatever their lengths.
enum DecodeQ8Mode { DQ_SLICE = 0, DQ_CLUSTER = 1, DQ_EVEN = 2 };

// DQ_EVEN: every slice is cut into chunks of at most `unit` blocks of keys, all of one size or one block apart, in the order of the slices; unit is
// the least for which `shares` blocks of threads are enough whatever the lengths.  Every warp works it out, two sequences a lane.
struct Cuts {
    int len[2], n[2], end[2];                                    // keys; chunks of each of its slices; chunks of all slices up to its last
    template <typename F>
    __device__ __forceinline__ Cuts(int B, int slices_each, int shares, F length) {
        const int lane = threadIdx.x & 31;
        int all = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            len[i] = lane + 32 * i < B ? length(lane + 32 * i) : 0;
            all += (len[i] + 31) / 32;
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
        const int rest = shares - B * slices_each, unit = max(1, (all * slices_each + rest - 1) / rest);
        int before = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            n[i] = ((len[i] + 31) / 32 + unit - 1) / unit;
            end[i] = n[i] * slices_each;
#pragma unroll
            for (int off = 1; off < 32; off *= 2) {
                const int up = __shfl_up_sync(0xffffffffu, end[i], off);
                if (lane >= off) end[i] += up;
            }
            end[i] += before;
            before = __shfl_sync(0xffffffffu, end[i], 31);
        }
    }
    // sequence of chunk c (B or more: there is none)
    __device__ __forceinline__ int sequence(int c) const {
        const int b = __popc(__ballot_sync(0xffffffffu, end[0] <= c)), more = __popc(__ballot_sync(0xffffffffu, end[1] <= c));
        return b < 32 ? b : 32 + more;
    }
    static __device__ __forceinline__ int of(const int (&x)[2], int b) { return __shfl_sync(0xffffffffu, b < 32 ? x[0] : x[1], b & 31); }
};

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

template <typename T, int DP, int NT, int MODE>
__global__ void __launch_bounds__(32 * DQ_WARPS, Shape<DP, NT>::ON_AN_SM)
decode_q8_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const DecodeQ8Params p) {
    decode_q8_prologue<DP, NT>(&tmap_k, &tmap_v);
    chain_wait();
    using S = Shape<DP, NT>;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int QP = F32 ? 2 : 1;                              // f16 parts of a value of q
    extern __shared__ __align__(1024) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int Hkv = p.H / p.G, R = p.G * p.Tq;
    const auto length = [&](int b) {
        const int len = p.lengths[b];
        if (len < 0 || len > p.cap) atomicCAS(p.told, 0u, (unsigned)DEERS_KERR_CACHE | 2u);
        return min(max(len, 0), p.cap);
    };
    if constexpr (MODE == DQ_CLUSTER) cooperative_groups::this_cluster().barrier_arrive();
    int stage = 0;                                               // of this warp's ring: where its next block is
    uint32_t phase = 0;
    int b, kvh, tile, len, blk0, blk1;
    bool whole = true;                                           // this block of threads sees all keys of the slice
    int chunks = 1;                                              // DQ_CLUSTER: blocks of threads that share them
    if constexpr (MODE == DQ_EVEN) {
        const Cuts cuts(p.B, Hkv * p.tiles, gridDim.x, length);
        b = cuts.sequence(blockIdx.x);
        if (b >= p.B) return;
        len = Cuts::of(cuts.len, b);
        const int n = Cuts::of(cuts.n, b), c = n * Hkv * p.tiles - (Cuts::of(cuts.end, b) - (int)blockIdx.x), slice = c / n, blocks = (len + 31) / 32;
        kvh = slice / p.tiles; tile = slice % p.tiles;
        blk0 = blocks * (c % n) / n;
        blk1 = blocks * (c % n + 1) / n;
        whole = n == 1;
    } else {
        b = blockIdx.y / Hkv; kvh = blockIdx.y % Hkv; tile = blockIdx.z;
    }
    const int row0 = tile * S::ROWS;
    // q is on its way while the length is (lane (g, t) has row g, channels 16 (t + 4 c) ..)
    alignas(16) T raw[NT][S::KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = row0 + nt * 8 + g;
        const T* src = static_cast<const T*>(p.q);
        if (r < R) src += b * p.sq[0] + (long long)(kvh * p.G + r / p.Tq) * p.sq[1] + (long long)(r % p.Tq) * p.sq[2];
#pragma unroll
        for (int i = 0; i < S::KS; i += 2) {                     // eight channels
            const int d = S::k_channel(i, t);
            const bool there = r < R && d < p.D;
            if (p.q_vec) {
#pragma unroll
                for (int w = 0; w < (int)sizeof(T) / 2; ++w)
                    reinterpret_cast<uint4*>(raw[nt][i])[w] = there ? reinterpret_cast<const uint4*>(src + d)[w] : make_uint4(0u, 0u, 0u, 0u);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) raw[nt][i + e / 4][e % 4] = there ? src[d + e] : T(0.f);
            }
        }
    }
    if constexpr (MODE != DQ_EVEN) {
        len = length(b);
        const int blocks = (len + 31) / 32, split = MODE == DQ_CLUSTER ? blockIdx.x : 0;
        if constexpr (MODE == DQ_CLUSTER) {
            // chunks have 256 keys or more: the cluster's other blocks leave (its barrier waits for those that stay; all have come to the first)
            chunks = max(1, min(p.splits, (blocks + 7) / 8));
            whole = chunks == 1;
            if (split >= chunks || whole) cooperative_groups::this_cluster().barrier_wait();
            if (split >= chunks) return;
        }
        blk0 = (int)((long long)blocks * split / chunks); blk1 = (int)((long long)blocks * (split + 1) / chunks);
    }
    const uint8_t* vb = p.v + b * p.sv[0] + kvh * p.sv[1];
    const float* ksl = p.k_scale + b * p.skl[0] + kvh * p.skl[1];
    const float* vsl = p.v_scale + b * p.svl[0] + kvh * p.svl[1];

    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::BARS) + warp * S::STAGES;
    const sm100::WaitState ws{reinterpret_cast<uint32_t*>(smem + S::BARS + DQ_WARPS * S::STAGES * 8), p.err};
    __syncthreads();                                             // the barriers are there
    uint8_t* ring = smem + warp * (S::STAGES * S::STAGE_BYTES);
    // Block `blk` into stage s, by one lane.  (Keys behind the sequence's last may lie in it, and are masked below.)
    auto fetch = [&](int blk, int s) {
        if (blk < blk1 && lane == 0) {
            sm100::mbar_arrive_expect_tx(&full[s], S::STAGE_BYTES);
#pragma unroll
            for (int i = 0; i < S::BOXES; ++i) {
                sm100::tma_load_4d(ring + s * S::STAGE_BYTES + i * 32 * S::BOX, &tmap_k, &full[s], i * S::BOX, blk * 32, kvh, b);
                sm100::tma_load_4d(ring + s * S::STAGE_BYTES + S::HALF_STAGE + i * 32 * S::BOX, &tmap_v, &full[s], i * S::BOX, blk * 32, kvh, b);
            }
        }
    };
    // Place of channel d of key j inside the boxes of K or of V (16-byte pieces lie swizzled)
    auto in_boxes = [&](int j, int d) {
        if constexpr (S::BOX == 64) return j * 64 + (((d >> 4) ^ (j >> 1 & 3)) << 4) + (d & 15);
        else return (d >> 7) * (32 * 128) + j * 128 + ((((d >> 4) & 7) ^ (j & 7)) << 4) + (d & 15);
    };
    // This lane's keys of a block: 8 r + g of K; 2t, 2t + 1, 2t + 8, 2t + 9 of either half of V.
    const auto v_key = [&](int r) { return (r >> 2) * 16 + ((r >> 1) & 1) * 8 + 2 * t + (r & 1); };
    const auto v_piece = [&](const uint8_t* st, int r, int d, auto& w) {
        const uint8_t* at = st + S::HALF_STAGE + in_boxes(v_key(r), d);
        if constexpr (sizeof(w) == 16) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(at);
        else if constexpr (sizeof(w) == 8) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(at);
        else w[0] = *reinterpret_cast<const uint32_t*>(at);
    };
    const auto k_words = [&](const uint8_t* st, int j, uint32_t (&w)[S::KS]) {
#pragma unroll
        for (int c = 0; c < S::KC; ++c) *reinterpret_cast<uint4*>(w + 4 * c) = *reinterpret_cast<const uint4*>(st + in_boxes(j, 16 * (t + 4 * c)));
        if constexpr (S::TAIL) *reinterpret_cast<uint2*>(w + 4 * S::KC) = *reinterpret_cast<const uint2*>(st + in_boxes(j, DP - 32 + 8 * t));
    };
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; ++s) fetch(blk0 + warp + s * DQ_WARPS, (stage + s) % S::STAGES);

    float ks_next = 0.f, vs_next = 0.f;                          // scales of the next round's block
    if (blk0 + warp < blk1) { ks_next = ksl[blk0 + warp]; vs_next = vsl[blk0 + warp]; }

    // q as the products' second operand
    uint32_t qf[NT][QP][S::KS][2];
    float qs[NT][2];                                             // factor of the scores of rows 2t, 2t + 1
    int lim[NT][2];                                              // keys that they see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float back = 1.f, up = 1.f;
        if constexpr (F32) {
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < S::KS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint((float)raw[nt][i][e]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // a power of two that brings the largest value to 2^14 .. 2^15 (exponents of factor and inverse both in range)
            int e = 141 - (int)(top >> 23);
            e = top == 0 || top >= 0x7f800000u ? 0 : min(100, e);       // (-113 or more)
            up = __uint_as_float((unsigned)(127 + e) << 23);
            back = __uint_as_float((unsigned)(127 - e) << 23);
        }
#pragma unroll
        for (int i = 0; i < S::KS; ++i)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float x = (float)raw[nt][i][2 * w] * up, y = (float)raw[nt][i][2 * w + 1] * up;
                qf[nt][0][i][w] = pack2(x, y);
                if constexpr (F32) {
                    const float2 hi = unpack2(qf[nt][0][i][w]);
                    qf[nt][1][i][w] = pack2(x - hi.x, y - hi.y);
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

    float o[NT][S::VT][4], m[NT][2], l[NT][2], most[NT][2];      // most: log2 of the largest weight times scale, no less than it is
    int up[NT][2];                                               // O is held times 2^up
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < S::VT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][j][e] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
        most[nt][0] = most[nt][1] = -INFINITY;
        up[nt][0] = up[nt][1] = 0;
    }

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
            constexpr int CHAINS = F32 ? (S::KS + 3) / 4 + 1 : 1;
            float sum[NT][CHAINS][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < CHAINS; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[nt][i][e] = 0.f;
            uint32_t xw[S::KS], yw[S::KS];
            k_words(st, 16 * mt + g, xw);
            k_words(st, 16 * mt + 8 + g, yw);
#pragma unroll
            for (int i = 0; i < S::KS; ++i) {
                const uint32_t a0 = q8::e4m3_lo(xw[i]), a2 = q8::e4m3_hi(xw[i]), a1 = q8::e4m3_lo(yw[i]), a3 = q8::e4m3_hi(yw[i]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816(sum[nt][F32 ? i / 4 : 0], a0, a1, a2, a3, qf[nt][0][i][0], qf[nt][0][i][1]);
                    if constexpr (F32) mma16816(sum[nt][CHAINS - 1], a0, a1, a2, a3, qf[nt][1][i][0], qf[nt][1][i][1]);
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
        const float vtop = (float)((int)(__float_as_uint(vs) >> 23 & 0xffu) - 126);      // vs < 2^vtop
        bool moved = false;
        float ofac[NT][2], vw[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float f = qs[nt][x] * ks;
                float here = -INFINITY;                          // the block's maximum
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
                    for (int y = 0; y < 2; ++y) here = fmaxf(here, s[nt][mt][2 * y + x]);
#pragma unroll
                for (int off = 4; off <= 16; off *= 2) here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, off));
                const float mx = fmaxf(m[nt][x], here);
                // (-inf: nothing seen so far, or NaN alone, which have to reach the sums)
                const float ms = mx == -INFINITY ? 0.f : mx, fac = power2(m[nt][x] - ms);
                m[nt][x] = mx;
                l[nt][x] *= fac;
                // Weights below 2^-110 count as 2^-110 here, so that 2^up stays in range.  (What fac makes zero of is no measure for the rest.)
                const bool seen = here > -INFINITY;
                most[nt][x] = fmaxf(fac > 0.f ? most[nt][x] : -INFINITY, seen ? fmaxf(here, ms - 110.f) + vtop : -INFINITY);
                const int to = DQ_UP - __float2int_ru(fmaxf(most[nt][x] - ms, -111.f));      // -114 to 126
                ofac[nt][x] = fac * power2_of(min(max(to - up[nt][x], -126), 127));
                vw[nt][x] = seen ? vs * power2_of(to) : 0.f;     // (a scale of any size where nothing is seen)
                up[nt][x] = to;
                moved |= ofac[nt][x] != 1.f;
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
                for (int j = 0; j < S::VT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[nt][j][e] *= ofac[nt][e & 1];
        }
        // ---- weights, transposed
        uint32_t pw[NT][2][2][2];                                // [tile][16 keys][part][8 keys]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float w0 = s[nt][mt][2 * y] * vw[nt][0], w1 = s[nt][mt][2 * y + 1] * vw[nt][1];
                    const uint32_t hi = pack2(w0, w1);
                    const float2 h = unpack2(hi);
                    pw[nt][mt][0][y] = transposed(hi);
                    pw[nt][mt][1][y] = transposed(pack2(w0 - h.x, w1 - h.y));
                }
        // A weight of zero does not keep out a NaN: where a key that some rows do not see holds one, the rows' sums are made one by one.
        if (edge && lim_min < len) {
            uint32_t nan = 0;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (v_key(r) >= len - blk * 32) continue;
                const auto look = [&](auto words, int d) {
                    uint32_t x[decltype(words)::value];
                    v_piece(st, r, d, x);
#pragma unroll
                    for (int w = 0; w < decltype(words)::value; ++w) nan |= ((x[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                };
#pragma unroll
                for (int c = 0; c < S::VC; ++c) look(std::integral_constant<int, S::VB / 4>(), S::VB * (g + 8 * c));
                if constexpr (S::TAIL) look(std::integral_constant<int, 1>(), DP - 32 + 4 * g);
            }
            if (__any_sync(0xffffffffu, nan != 0)) {
                if constexpr (F32) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < S::VT; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nt][j][e] *= ofac[nt][e & 1];
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
                                for (int x = 0; x < 2; ++x) w[x] = __shfl_sync(0xffffffffu, s[nt][mt][2 * y + x], i * 4 + t) * vw[nt][x];
#pragma unroll
                                for (int j = 0; j < S::VT; ++j) {
                                    const int d = S::v_channel(j, g);
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
        // one piece of the channels of all 32 keys at a time
        const int behind = len - blk * 32;
        const auto tiles = [&](auto words, int j0, int d) {      // words of a key's piece, its first tile and channel
            constexpr int W = decltype(words)::value;
            uint32_t x[8][W];
#pragma unroll
            for (int r = 0; r < 8; ++r) v_piece(st, r, d, x[r]);
            if (behind < 32) {                                   // what lies behind the last key is nobody's, and may be NaN
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (v_key(r) >= behind) {
#pragma unroll
                        for (int w = 0; w < W; ++w) x[r][w] = 0;
                    }
            }
#pragma unroll
            for (int jj = 0; jj < 2 * W; ++jj) {
                uint32_t a[2][4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t e0 = __byte_perm(x[4 * h][jj / 2], x[4 * h + 1][jj / 2], jj & 1 ? 0x7362 : 0x5140);
                    const uint32_t e1 = __byte_perm(x[4 * h + 2][jj / 2], x[4 * h + 3][jj / 2], jj & 1 ? 0x7362 : 0x5140);
                    a[h][0] = q8::e4m3_lo(e0); a[h][1] = q8::e4m3_hi(e0); a[h][2] = q8::e4m3_lo(e1); a[h][3] = q8::e4m3_hi(e1);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float (&to)[4] = o[nt][j0 + jj];
                    if constexpr (F32) {
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int part = 1; part >= 0; --part)
#pragma unroll
                            for (int h = 0; h < 2; ++h) mma16816(sum, a[h][0], a[h][1], a[h][2], a[h][3], pw[nt][h][part][0], pw[nt][h][part][1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) to[e] = fmaf(to[e], ofac[nt][e & 1], sum[e]);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int part = 0; part < 2; ++part) mma16816(to, a[h][0], a[h][1], a[h][2], a[h][3], pw[nt][h][part][0], pw[nt][h][part][1]);
                    }
                }
            }
        };
#pragma unroll
        for (int c = 0; c < S::VC; ++c) tiles(std::integral_constant<int, S::VB / 4>(), c * (S::VB / 2), S::VB * (g + 8 * c));
        if constexpr (S::TAIL) tiles(std::integral_constant<int, 1>(), S::VT - 2, DP - 32 + 4 * g);
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
    {
        float* mine = meet + warp * S::ROWS * S::OS;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float down[2] = {power2_of(-up[nt][0]), power2_of(-up[nt][1])};
#pragma unroll
            for (int j = 0; j < S::VT; ++j) {
                const int d = S::v_channel(j, g);
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[(nt * 8 + 2 * t + (e & 1)) * S::OS + d + (e >> 1)] = o[nt][j][e] * down[e & 1];
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
    const auto finish = [&](int r, int d, const float4& v, float mx, float sum) {      // four channels of a row
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        put4(out_row(r) + d, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv), p.o_vec);
        if (p.lse && d == 0) *lse_at(r) = (mx + log2f(sum)) * DQ_LN2;
    };
    float* to_part = p.part + (long long)blockIdx.x * (S::ROWS * (p.D + 4));      // DQ_EVEN
    const int share = ((rows * p.D + chunks - 1) / chunks + 3) / 4 * 4;             // DQ_CLUSTER: of the outputs, to every block
    if (MODE == DQ_CLUSTER && !whole) cooperative_groups::this_cluster().barrier_wait();       // (all have started: their memory may be written to)
    for (int r = warp; r < rows; r += DQ_WARPS) {
        float w[DQ_WARPS], mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int x = 0; x < DQ_WARPS; ++x) {
            w[x] = meet[(x * S::ROWS + r) * S::OS + DP];
            mx = fmaxf(mx, w[x]);
        }
        const float ms = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int x = 0; x < DQ_WARPS; ++x) {
            w[x] = exp2f(w[x] - ms);
            sum = fmaf(w[x], meet[(x * S::ROWS + r) * S::OS + DP + 1], sum);
        }
        for (int d = 4 * lane; d < p.D; d += 128) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < DQ_WARPS; ++x) add4(v, w[x], *reinterpret_cast<const float4*>(&meet[(x * S::ROWS + r) * S::OS + d]));
            if (MODE == DQ_CLUSTER && !whole) {
                const int i = r * p.D + d, z = i / share;
                const uint32_t to = sm100::cluster_addr(smem + S::SENT, z);
                send4(to + 8 * 8 * S::ROWS + 4 * (blockIdx.x * share + i - z * share), v);
                // (whoever owns channels of a row needs its maxima and sums: the first of its channels, or of that share, brings them)
                if (d == 0 || i == z * share) {
                    send(to + 8 * (blockIdx.x * S::ROWS + r), mx);
                    send(to + 8 * (blockIdx.x * S::ROWS + r) + 4, sum);
                }
            } else if (MODE == DQ_SLICE || whole) {
                finish(r, d, v, mx, sum);
            } else {
                *reinterpret_cast<float4*>(to_part + r * (p.D + 4) + d) = v;
                if (d == 0) *reinterpret_cast<float2*>(to_part + r * (p.D + 4) + p.D) = make_float2(mx, sum);
            }
        }
    }
    if (MODE == DQ_CLUSTER && !whole) {
        cooperative_groups::this_cluster().sync();
        const float2* ml = reinterpret_cast<const float2*>(smem + S::SENT);
        const float* parts = reinterpret_cast<const float*>(ml + 8 * S::ROWS);
        const int end = min(share, rows * p.D - (int)blockIdx.x * share);
        for (int j = 4 * (int)threadIdx.x; j < end; j += 128 * DQ_WARPS) {
            const int i = blockIdx.x * share + j, r = i / p.D;
            float w[8], mx = -INFINITY, sum = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                w[z] = z < chunks ? ml[z * S::ROWS + r].x : -INFINITY;
                mx = fmaxf(mx, w[z]);
            }
            const float ms = mx == -INFINITY ? 0.f : mx;
#pragma unroll
            for (int z = 0; z < 8; ++z)
                if (z < chunks) {
                    const float f = exp2f(w[z] - ms);
                    sum = fmaf(f, ml[z * S::ROWS + r].y, sum);
                    add4(v, f, *reinterpret_cast<const float4*>(&parts[z * share + j]));
                }
            finish(r, i - r * p.D, v, mx, sum);
        }
    }
}

// Rows of slices that no block of threads has seen whole, from what each has left of them; one row a block.
template <typename T>
__global__ void __launch_bounds__(256) decode_q8_join_kernel(const DecodeQ8Params p, int tile_rows, int shares) {
    chain_wait();
    __shared__ float s_w[DQ_MAX_SHARES], s_l[DQ_MAX_SHARES], s_r[16];
    __shared__ __align__(16) float s_o[8][256];
    const int r = blockIdx.x, tile = blockIdx.z, Hkv = p.H / p.G, b = blockIdx.y / Hkv, kvh = blockIdx.y % Hkv;
    const int rr = tile * tile_rows + r, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (rr >= p.G * p.Tq) return;
    const Cuts cuts(p.B, Hkv * p.tiles, shares, [&](int x) { return min(max(p.lengths[x], 0), p.cap); });
    const int n = Cuts::of(cuts.n, b), first = Cuts::of(cuts.end, b) - n * (Hkv * p.tiles - kvh * p.tiles - tile);
    if (n == 1) return;                                          // seen whole
    const int head = kvh * p.G + rr / p.Tq, i = rr % p.Tq;
    T* o = static_cast<T*>(p.o) + b * p.so[0] + head * p.so[1] + i * p.so[2];
    float* lse = p.lse ? p.lse + ((long long)b * p.H + head) * p.Tq + i : nullptr;
    if (n == 0) {                                                // a sequence without keys is nobody's share
        for (int d = threadIdx.x; d < p.D; d += 256) put(o + d, 0.f);
        if (lse && threadIdx.x == 0) *lse = -INFINITY;
        return;
    }
    const int step = tile_rows * (p.D + 4);
    const float* part = p.part + (long long)first * step + r * (p.D + 4);
    float mx = -INFINITY;
    for (int z = threadIdx.x; z < n; z += 256) {
        const float2 ms = *reinterpret_cast<const float2*>(part + z * step + p.D);
        s_w[z] = ms.x; s_l[z] = ms.y;
        mx = fmaxf(mx, ms.x);
    }
    // (what the first turn below wants is on its way meanwhile)
    float4 early[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        early[i] = warp + 8 * i < n && 4 * lane < p.D ? *reinterpret_cast<const float4*>(part + (warp + 8 * i) * step + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
    if (lane == 0) s_r[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = fmaxf(mx, s_r[w]);
    const float ms = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    for (int z = threadIdx.x; z < n; z += 256) {
        const float w = exp2f(s_w[z] - ms);
        s_w[z] = w;
        sum = fmaf(w, s_l[z], sum);
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (lane == 0) s_r[8 + warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += s_r[8 + w];
    // a warp adds up every eighth chunk, four channels a lane
    for (int d = 4 * lane; d < p.D; d += 128) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        int z = warp;
        if (d < 128) {
#pragma unroll
            for (int i = 0; i < 4; ++i, z += 8)
                if (z < n) add4(v, s_w[z], early[i]);
        }
#pragma unroll 4
        for (; z < n; z += 8) add4(v, s_w[z], *reinterpret_cast<const float4*>(part + z * step + d));
        *reinterpret_cast<float4*>(&s_o[warp][d]) = v;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += 256) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += s_o[w][d];
        put(o + d, sum == 0.f ? 0.f : v / sum);
    }
    if (lse && threadIdx.x == 0) *lse = (mx + log2f(sum)) * DQ_LN2;
}

struct DecodeQ8Plan { int dp, nt, tiles, mode, splits, shares; };   // splits: blocks of a cluster; shares: of all blocks

// How the work is cut.  Sixteen query rows share a walk where there are more than eight (heads up to 128 wide: the registers hold their O).
// The host knows how many keys a slice can hold, not how many it holds.  Each slice gets as many blocks of threads (a cluster, 8 at most) as put
// two on every SM, or seven where slices are long: ragged lengths then leave less of the device idle at the end (512 slices of 16384 keys, f16,
// D = 128, lengths uniform from 0 / all full: 2 blocks 188 / 350 us, 1 block 225 / 472).  Blocks whose lengths leave them less than 256 keys go
// again at once.  Few long slices are cut on the device in proportion to their keys, for a second launch (against 8 blocks a slice): 16 slices of
// 65536 keys 31 / 49 us against 61 / 93, 64 of 16384 33 / 52 against 43 / 67, 16 of 16384 13 / 20 against 18 / 27.  Shorter ones gain nothing
// (32 of 8192 keys 15 / 20 against 15 / 19; 32 of 4096 13 / 15 against 12 / 14).
// From 65 slices on, and below 16384 keys, the cut goes by the capacity, so ragged lengths leave SMs idle: f16, D = 128, uniform from 0 / all full, of
// the copy rate: 16 x 8 slices of 4096 keys, G 4, 25 / 31 us (0.44 / 0.67); 10 x 32 of 2048 23 / 33 (0.51 / 0.79); 16 x 32 of 2048 33 / 58 (0.57 / 0.71);
// 40 x 8 of 4096 54 / 59 (0.51 / 0.88); 64 x 8 of 2048, G 4, 34 / 59 (0.55 / 0.71), of 8192 91 / 205 (0.76 / 0.81).
// (148: the SMs of a B200.  The workspace's size is asked for without a context.)
DecodeQ8Plan plan_decode_q8(const deers_decode_q8_desc* d) {
    DecodeQ8Plan p;
    p.dp = d->cache.D > 128 ? 256 : (d->cache.D + 31) / 32 * 32;
    const int R = d->H / d->cache.H * d->Tq;
    p.nt = R > 8 && p.dp <= 128 ? 2 : 1;
    p.tiles = (R + 8 * p.nt - 1) / (8 * p.nt);
    const long long slices = (long long)d->cache.B * d->cache.H * p.tiles;
    const long long blocks = (d->cache.capacity + 31) / 32;
    p.mode = DQ_SLICE; p.splits = 1; p.shares = 0;
    if (d->cache.capacity >= DQ_LONG && slices <= DQ_MAX_EVEN) {
        const long long most = slices * blocks / 14, fill = p.dp > 128 ? DQ_MAX_SHARES / 2 : DQ_MAX_SHARES;      // (heads of 256: one block of threads an SM)
        p.mode = DQ_EVEN;
        p.shares = (int)(most < fill ? most : fill);
    } else {
        long long want = (d->cache.capacity >= DQ_LONG ? 7 * 148 : 2 * 148) / slices;
        const long long most = (blocks + 7) / 8;                 // at least 256 keys a chunk
        if (want > most) want = most;
        if (want > 8) want = 8;
        if (want > 1) { p.mode = DQ_CLUSTER; p.splits = (int)want; }
    }
    return p;
}

size_t decode_q8_bytes(const deers_decode_q8_desc* d, const DecodeQ8Plan& p) {
    if (p.mode != DQ_EVEN) return 0;
    return (size_t)p.shares * (8 * p.nt) * (d->cache.D + 4) * sizeof(float);
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
    if (plan.mode == DQ_SLICE) {
        DEERS_SMEM_ONCE(ctx, (decode_q8_kernel<T, DP, NT, DQ_SLICE>), S::SMEM);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_kernel<T, DP, NT, DQ_SLICE>, dim3(1, slices, plan.tiles), 32 * DQ_WARPS, S::SMEM, 1, tk, tv, p));
    } else if (plan.mode == DQ_CLUSTER) {
        DEERS_SMEM_ONCE(ctx, (decode_q8_kernel<T, DP, NT, DQ_CLUSTER>), S::SMEM);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_kernel<T, DP, NT, DQ_CLUSTER>, dim3(plan.splits, slices, plan.tiles), 32 * DQ_WARPS, S::SMEM, plan.splits, tk, tv, p));
    } else {
        DEERS_SMEM_ONCE(ctx, (decode_q8_kernel<T, DP, NT, DQ_EVEN>), S::SMEM);
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_kernel<T, DP, NT, DQ_EVEN>, (unsigned)plan.shares, 32 * DQ_WARPS, S::SMEM, 1, tk, tv, p));
        DEERS_CUDA_TRY(ctx, launch_chained(ctx, decode_q8_join_kernel<T>, dim3(S::ROWS, slices, plan.tiles), 256, 0, 1, p, S::ROWS, plan.shares));
        ctx->launches += 1;
    }
    return DEERS_OK;
}

template <typename T>
int decode_q8_widths(deers_ctx* ctx, const DecodeQ8Params& p, const DecodeQ8Plan& plan, int slices, const deers_cache_q8& c) {
    switch (plan.dp) {
        case 32: return plan.nt == 2 ? decode_q8_launch<T, 32, 2>(ctx, p, plan, slices, c) : decode_q8_launch<T, 32, 1>(ctx, p, plan, slices, c);
        case 64: return plan.nt == 2 ? decode_q8_launch<T, 64, 2>(ctx, p, plan, slices, c) : decode_q8_launch<T, 64, 1>(ctx, p, plan, slices, c);
        case 96: return plan.nt == 2 ? decode_q8_launch<T, 96, 2>(ctx, p, plan, slices, c) : decode_q8_launch<T, 96, 1>(ctx, p, plan, slices, c);
        case 128: return plan.nt == 2 ? decode_q8_launch<T, 128, 2>(ctx, p, plan, slices, c) : decode_q8_launch<T, 128, 1>(ctx, p, plan, slices, c);
        default: break;
    }
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
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15u))) return DEERS_ERR_WORKSPACE;
    DEERS_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    const deers_cache_q8& c = d->cache;
    DecodeQ8Params p;
    p.q = q; p.o = o; p.lse = lse; p.lengths = lengths;
    p.part = need ? (float*)workspace : nullptr;
    p.k = (const uint8_t*)c.k; p.v = (const uint8_t*)c.v; p.k_scale = c.k_scale; p.v_scale = c.v_scale;
    for (int i = 0; i < 3; ++i) { p.sq[i] = d->q_strides[i]; p.so[i] = d->o_strides[i]; p.sk[i] = c.k_strides[i]; p.sv[i] = c.v_strides[i]; }
    for (int i = 0; i < 2; ++i) { p.skl[i] = c.k_scale_strides[i]; p.svl[i] = c.v_scale_strides[i]; }
    p.B = c.B; p.tiles = plan.tiles;
    p.H = d->H; p.G = d->H / c.H; p.Tq = d->Tq; p.D = c.D; p.cap = c.capacity; p.causal = d->causal; p.splits = plan.splits;
    p.scale = d->scale; p.err = ctx->dev_err; p.told = ctx->dev_err + 1;
    const int64_t al = 16 / (int64_t)es - 1;
    p.o_vec = ((uintptr_t)o & 15u) == 0 && ((d->o_strides[0] | d->o_strides[1] | d->o_strides[2]) & al) == 0;
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
