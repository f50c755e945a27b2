// Rows of activations as 8-bit codes with a scale each: what the 8-bit products read (gemm_q8_sm100.cu).
//
//     h = x + residual (rounded to the stream's type and written), or x, or max(x, 0)^2
//     y = h / sqrt(mean(h * h) + eps), or h
//     scale = max|y| / Q,  code = nearest(y / scale)           Q = 127 (int8) or 448 (e4m3)
//
// The norm is one factor per row, so it cancels in the codes: code = nearest(h * Q / max|h|), and only the scale carries it.  One pass over
// the row (its maximum and its sum of squares meet in one exchange), codes from the registers that hold it; the norm's rows in f32 and the
// pass that would quantise them never exist.  Codes are the nearest to the exact quotient (q8_codes.cuh).
// Squares of f32 values beyond 2^48 or below 2^-40 may leave f32: the sum of such a row is made again in 64 bits, from memory (in front of the codes; at the
// kernel's end it costs every row 4 to 11 %, three sums of scaled squares as much, this 0 to 3).
// A row of zeros has scale 0.  A row with an infinity or a NaN has scale NaN and codes 0: every product of it is NaN, as it is of the norm.
// Bound: HBM, 7 bytes an element with f16 and a residual, 13 with f32: 16384 x 2048 f16 42 us (int8; e4m3 41, 0.88 of the copy rate), 8192 x 4096 f32 80 (78, 0.86).
// Rows on smaller boundaries move fewer bytes an access, codes as few at a time as values: f16 4096 x 4100 39 us (8 bytes; 0.47), 8192 x 2731 68 to 72 (2 bytes; 0.35),
// f32 5000 x 1025 15 (4 bytes; 0.68).  Rows longer than registers hold are read twice: f32 3000 x 12000 102 to 104 (0.70), f16 2000 x 20000 68 to 70 (0.63).
// relu^2 reads a third of the bytes and is bound by instructions: f16 16384 x 2048 28.5 us (0.55).
// What it took: a row on as few threads as hold it in 40 registers, so that an SM has 1536 (48 -> 42 us; at 60 registers loads of too few rows
// were in flight); borders between codes decided by exact products instead of a 64-bit division for every value next to one (relative to
// that 51 -> 48, and new keys and values, cache_q8.cu, 141 -> 43, by remainders of f16 quotients 42.0 -> 41.3); units that neighbouring threads interleave where rows start on no 16-byte
// boundary (4096 x 4100 f16 106 -> 39 us).
#include "common.cuh"
#include "q8_codes.cuh"

namespace {

struct QuantParams {
    const void* x; const void* residual; void* sum; uint8_t* codes; float* scale;
    long long ld_x, ld_res, ld_sum, ld_codes;
    long long rows;
    int C;
    float eps, inv_n;
    int norm;
};

__device__ __forceinline__ void from_f(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
template <int N>
__device__ __forceinline__ void add_to(float (&v)[N], const float (&r)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += r[e];
}
template <int N>
__device__ __forceinline__ void add_to(__half (&v)[N], const __half (&r)[N]) {                  // (rounded once)
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const __half2 s = __hadd2_rn(__halves2half2(v[e], v[e + 1]), __halves2half2(r[e], r[e + 1]));
        v[e] = __low2half(s);
        v[e + 1] = __high2half(s);
    }
}
__device__ __forceinline__ float squared_relu(float v) { return v <= 0.f ? 0.f : v * v; }      // (a NaN stays one)

// U elements (a unit, one access): 16 bytes where rows allow, less where they start on smaller boundaries.
template <int BYTES> struct Word;
template <> struct Word<16> { typedef uint4 type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<4> { typedef uint32_t type; };
template <> struct Word<2> { typedef uint16_t type; };
template <> struct Word<1> { typedef uint8_t type; };
template <typename T, int U>
__device__ __forceinline__ void load_unit(const T* p, int n, T* v) {
    typedef typename Word<U * (int)sizeof(T)>::type W;
    if (U == 1 || n >= U) {
        *reinterpret_cast<W*>(v) = *reinterpret_cast<const W*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < U; ++e) {
            from_f(v[e], 0.f);
            if (e < n) v[e] = p[e];
        }
    }
}
template <typename T, int U>
__device__ __forceinline__ void store_unit(T* p, int n, const T* v) {
    typedef typename Word<U * (int)sizeof(T)>::type W;
    if (U == 1 || n >= U) {
        *reinterpret_cast<W*>(p) = *reinterpret_cast<const W*>(v);
    } else {
#pragma unroll
        for (int e = 0; e < U; ++e)
            if (e < n) p[e] = v[e];
    }
}

// top / sqrt(mean(h * h) + eps) of an f32 row in 64 bits, by the tpr threads that share it; read again, which keeps the registers of the rows that do without.
// 0 where 32 bits do, or there is nothing to divide: what squares lose above 2^-40 is less than 2^-40 of their sum, and an eps of 2^-50 outweighs those below.
static __device__ __noinline__ float norm64(const float* x, const float* residual, int C, float top, float eps, int tid, int tpr) {
    if (!(top > 0.f && top < __uint_as_float(0x7f800000u)) || (top < 1.f && eps >= 8.8817842e-16f)) return 0.f;
    __shared__ double s_d[16];
    double d = 0.0;
    for (int at = tid; at < C; at += tpr) {
        const double h = residual ? x[at] + residual[at] : x[at];
        d = fma(h, h, d);
    }
    for (int off = 16; off >= 1; off >>= 1) d += __shfl_xor_sync(0xffffffffu, d, off);
    if (tpr > 32) {
        if ((tid & 31) == 0) s_d[tid >> 5] = d;
        __syncthreads();
        d = 0.0;
        for (int w = 0; w < tpr / 32; ++w) d += s_d[w];
    }
    return (float)((double)top / sqrt(d / C + eps));
}

// TPR threads share a row (32: a warp, eight rows a block; else the block).  A thread holds NP pieces of N elements in registers, a piece being
// N / U units that neighbouring threads interleave, so that every access of a warp is contiguous.  NP = 0: rows of any length, read again
// for their codes.
template <typename T, bool I8, bool RELU2, int U, int TPR, int NP>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, NP > 0 ? 1536 / (TPR == 32 ? 256 : TPR) : 1) quantize_rows_kernel(const QuantParams p) {
    chain_wait();
    constexpr int N = U > 4 ? U : 4, UNITS = N / U;              // elements of a piece, units of it
    constexpr float MOST = I8 ? q8::MOST_I8 : q8::MOST_E4M3;
    const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5;
    const long long row = TPR == 32 ? (long long)blockIdx.x * 8 + warp : (long long)blockIdx.x;
    if (row >= p.rows) return;                                   // (a warp's own row: no block barrier with TPR == 32)
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ld_res : nullptr;
    T* sum = p.sum ? static_cast<T*>(p.sum) + row * p.ld_sum : nullptr;
    uint8_t* codes = p.codes + row * p.ld_codes;
    float top = 0.f, ss = 0.f;                                   // max|h| (of the numbers; a NaN is in the sum) and sum h^2
    const auto place = [&](int piece, int unit) { return ((piece * UNITS + unit) * TPR + tid) * U; };
    const auto has = [&](int piece) { return place(piece, 0) < p.C; };

    auto fetch = [&](int piece, T (&v)[N]) {                     // h; zeros behind the row's end
        T r[N];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int at = place(piece, u);
#pragma unroll
            for (int e = 0; e < U; ++e) { from_f(v[u * U + e], 0.f); from_f(r[u * U + e], 0.f); }
            if (at < p.C) {
                load_unit<T, U>(x + at, p.C - at, v + u * U);
                if (res) load_unit<T, U>(res + at, p.C - at, r + u * U);
            }
        }
        if (res) add_to(v, r);
    };
    auto values = [&](const T (&v)[N], int e, float (&f)[4]) {
        q8::four(v + e, f);
        if constexpr (RELU2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = squared_relu(f[k]);
        }
    };
    auto look = [&](const T (&v)[N]) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            float f[4];
            values(v, e, f);
            q8::look_at(top, f);
#pragma unroll
            for (int k = 0; k < 4; ++k) ss = fmaf(f[k], f[k], ss);
        }
    };
    alignas(16) T v[NP ? NP : 1][N];
    if constexpr (NP > 0) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (has(i)) fetch(i, v[i]);
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (has(i)) look(v[i]);
    } else {
#pragma unroll 1
        for (int i = 0; has(i); ++i) {
            fetch(i, v[0]);
            look(v[0]);
        }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        ss += __shfl_xor_sync(0xffffffffu, ss, off);
    }
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        __shared__ float s_top[W], s_ss[W];
        if ((threadIdx.x & 31) == 0) { s_top[warp] = top; s_ss[warp] = ss; }
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { top = fmaxf(top, s_top[w]); ss += s_ss[w]; }
    }
    const bool number = top < __uint_as_float(0x7f800000u) && ss == ss, some = number && top > 0.f;
    float far = 0.f;
    if constexpr (sizeof(T) == 4 && !RELU2) {
        // squares of values beyond 2^48, in rows of up to 2^30, may leave f32, and so may those below 2^-40 (the row's threads agree)
        if (__builtin_expect(p.norm && !(top > 9.0949470e-13f && top < 2.8147498e14f), 0)) far = norm64(x, res, p.C, top, p.eps, tid, TPR);
    }
    if (tid == 0) {
        float s = top;
        if (p.norm) s = top * (1.0f / sqrtf(ss * p.inv_n + p.eps));
        if (sizeof(T) == 4 && far > 0.f) s = far;
        p.scale[row] = !number ? __uint_as_float(0x7fc00000u) : some ? s / MOST : 0.f;
    }
    const q8::Factors factors = q8::factors(MOST, top, q8::den_is_far(top));
    auto put = [&](int piece, const T (&v)[N]) {
        uint32_t c[N / 4];
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            float f[4];
            values(v, e, f);
            c[e / 4] = some ? q8::codes_of<I8, sizeof(T) == 2 && !RELU2>(f, factors, MOST, top) : 0u;      // (448 has three bits, an f16 value eleven)
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int at = place(piece, u);
            if (at < p.C) {                                      // rows of codes start on 16-byte boundaries
                if (sum) store_unit<T, U>(sum + at, p.C - at, v + u * U);
                store_unit<uint8_t, U>(codes + at, p.C - at, reinterpret_cast<const uint8_t*>(c) + u * U);
            }
        }
    };
    if constexpr (NP > 0) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (has(i)) put(i, v[i]);
    } else {
#pragma unroll 1
        for (int i = 0; has(i); ++i) {
            fetch(i, v[0]);
            put(i, v[0]);
        }
    }
    chain_next();                                                // (at the start, a product's few large blocks settle unevenly on the SMs that are free first: 20.8 us with it, 15)
}

template <typename T, bool I8, int U, bool RELU2>
int quant_widths(deers_ctx* ctx, const QuantParams& p) {
    constexpr int N = U > 4 ? U : 4;
    const int pieces = (p.C + N - 1) / N;
    KernelTimerScope ts(ctx, DEERS_K_NORM);
    const unsigned rows = (unsigned)p.rows;
#define DEERS_ROWS(TPR, NP) \
    DEERS_CUDA_TRY(ctx, launch_chained(ctx, quantize_rows_kernel<T, I8, RELU2, U, TPR, NP>, TPR == 32 ? (rows + 7) / 8 : rows, TPR == 32 ? 256 : TPR, 0, 1, p))
    if (pieces <= 32) DEERS_ROWS(32, 1);
    else if (pieces <= 64) DEERS_ROWS(32, 2);
    else if (pieces <= 256) DEERS_ROWS(128, 2);
    else if (pieces <= 512) DEERS_ROWS(256, 2);
    else if (pieces <= 1024) DEERS_ROWS(512, 2);
    else if (pieces <= 2048) DEERS_ROWS(512, 4);
    else DEERS_ROWS(512, 0);
#undef DEERS_ROWS
    return DEERS_OK;
}
template <typename T, bool I8, int U>
int quant_launch(deers_ctx* ctx, const QuantParams& p, bool relu2) {
    return relu2 ? quant_widths<T, I8, U, true>(ctx, p) : quant_widths<T, I8, U, false>(ctx, p);
}

}  // namespace

extern "C" int deers_b200_quantize_rows(deers_ctx* ctx, const deers_quantize_desc* d, const void* x, const void* residual, void* sum,
                                        void* codes, float* scale) {
    if (!ctx || !d) return DEERS_ERR_NULL;
    if (d->dtype != DEERS_F16 && d->dtype != DEERS_F32) return DEERS_ERR_DTYPE;
    if (d->code != DEERS_I8 && d->code != DEERS_E4M3) return DEERS_ERR_DTYPE;
    if (d->rows < 0 || d->rows > 0x7fffffffLL || d->C < 1) return DEERS_ERR_SHAPE;
    if (d->C > (1 << 30)) return DEERS_ERR_UNSUPPORTED;          // (places behind a row's end stay within 31 bits)
    if (d->relu_squared && (d->norm || residual || sum)) return DEERS_ERR_UNSUPPORTED;
    if (d->rows == 0) return DEERS_OK;
    if (!x || !codes || !scale || (residual && !sum)) return DEERS_ERR_NULL;
    if (sum && !residual) return DEERS_ERR_UNSUPPORTED;
    const uintptr_t es = d->dtype == DEERS_F16 ? 2 : 4;
    if (d->ld_x < 0 || d->ld_codes < d->C || (d->ld_codes & 15) || ((uintptr_t)codes & 15u) || ((uintptr_t)scale & 3u)) return DEERS_ERR_LAYOUT;
    if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum) & (es - 1)) return DEERS_ERR_LAYOUT;
    if (residual && (d->ld_residual < 0 || d->ld_sum < d->C)) return DEERS_ERR_LAYOUT;
    DEERS_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    QuantParams p;
    p.x = x; p.residual = residual; p.sum = sum; p.codes = (uint8_t*)codes; p.scale = scale;
    p.ld_x = d->ld_x; p.ld_res = residual ? d->ld_residual : 0; p.ld_sum = sum ? d->ld_sum : 0; p.ld_codes = d->ld_codes;
    p.rows = d->rows; p.C = d->C; p.eps = (float)d->eps; p.inv_n = (float)(1.0 / (double)d->C);
    p.norm = d->norm;
    const uintptr_t at = (uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum | (uintptr_t)((p.ld_x | p.ld_res | p.ld_sum) * (long long)es);
    const bool half = d->dtype == DEERS_F16, i8 = d->code == DEERS_I8, wide = (at & 15) == 0, half16 = (at & 7) == 0, pair = (at & 3) == 0;
    const auto go = half ? (i8 ? (wide ? quant_launch<__half, true, 8> : half16 ? quant_launch<__half, true, 4> : pair ? quant_launch<__half, true, 2> : quant_launch<__half, true, 1>)
                               : (wide ? quant_launch<__half, false, 8> : half16 ? quant_launch<__half, false, 4> : pair ? quant_launch<__half, false, 2> : quant_launch<__half, false, 1>))
                         : (i8 ? (wide ? quant_launch<float, true, 4> : half16 ? quant_launch<float, true, 2> : quant_launch<float, true, 1>)
                               : (wide ? quant_launch<float, false, 4> : half16 ? quant_launch<float, false, 2> : quant_launch<float, false, 1>));
    const int rc = go(ctx, p, d->relu_squared != 0);
    if (rc) return rc;
    ctx->launches += 1;
    DEERS_CUDA_TRY(ctx, cudaGetLastError());
    return DEERS_OK;
}
