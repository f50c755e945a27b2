// Rows of activations as 8-bit codes with a scale each: what the 8-bit products read (gemm_q8_sm100.cu).
//
//     h = x + residual (rounded to the stream's type and written), or x, or max(x, 0)^2
//     y = h / sqrt(mean(h * h) + eps), or h
//     scale = max|y| / Q,  code = nearest(y / scale)           Q = 127 (int8) or 448 (e4m3)
//
// The norm is one factor per row, so it cancels in the codes: code = nearest(h * Q / max|h|), and only the scale carries it.  One pass over
// the row (its maximum and its sum of squares meet in one exchange), codes from the registers that hold it; the norm's rows in f32 and the
// pass that would quantise them never exist.  Codes are the nearest to the exact quotient (q8_codes.cuh).
// A row of zeros has scale 0.  A row with an infinity or a NaN has scale NaN and codes 0: every product of it is NaN, as it is of the norm.
// Bound: HBM, 7 bytes an element with f16 and a residual, 13 with f32.
#include "common.cuh"
#include "q8_codes.cuh"

namespace {

struct QuantParams {
    const void* x; const void* residual; void* sum; uint8_t* codes; float* scale;
    long long ld_x, ld_res, ld_sum, ld_codes;
    long long rows;
    int C;
    float eps, inv_n;
    int norm, relu2;
};

template <typename T> struct Piece;                              // 16 bytes of a row
template <> struct Piece<__half> { static constexpr int N = 8; };
template <> struct Piece<float> { static constexpr int N = 4; };

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }

// n valid elements (0..N) at p; VEC: p lies on a 16-byte boundary.
template <typename T, bool VEC>
__device__ __forceinline__ void load_piece(const T* p, int n, T (&v)[Piece<T>::N]) {
    constexpr int N = Piece<T>::N;
    if (VEC && n == N) {
        *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            from_f(v[e], 0.f);
            if (e < n) v[e] = p[e];
        }
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_piece(T* p, int n, const T (&v)[Piece<T>::N]) {
    constexpr int N = Piece<T>::N;
    if (VEC && n == N) {
        *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < n) p[e] = v[e];
    }
}

__device__ __forceinline__ float squared_relu(float v) { return v <= 0.f ? 0.f : v * v; }      // (a NaN stays one)

// TPR threads share a row (32: a warp, eight rows a block; else the block), NP pieces each, which stay in registers.  NP = 0: rows of any
// length, read again for their codes.
template <typename T, bool I8, bool VEC, int TPR, int NP>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) quantize_rows_kernel(const QuantParams p) {
    chain_begin();
    constexpr int N = Piece<T>::N;
    constexpr float MOST = I8 ? q8::MOST_I8 : q8::MOST_E4M3;
    const int tid = TPR == 32 ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5;
    const long long row = TPR == 32 ? (long long)blockIdx.x * 8 + warp : (long long)blockIdx.x;
    if (row >= p.rows) return;                                   // (a warp's own row: no block barrier with TPR == 32)
    const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.ld_res : nullptr;
    T* sum = p.sum ? static_cast<T*>(p.sum) + row * p.ld_sum : nullptr;
    uint8_t* codes = p.codes + row * p.ld_codes;
    const int pieces = (p.C + N - 1) / N;
    unsigned top = 0;                                            // max|h| as bits: infinities and NaN order above all numbers
    float ss = 0.f;

    auto fetch = [&](int at, T (&v)[N]) {                        // h of piece `at`
        const int n = min(N, p.C - at * N);
        load_piece<T, VEC>(x + (long long)at * N, n, v);
        if (res) {
            T r[N];
            load_piece<T, VEC>(res + (long long)at * N, n, r);
#pragma unroll
            for (int e = 0; e < N; ++e) from_f(v[e], to_f(v[e]) + to_f(r[e]));
        }
    };
    auto look = [&](const T (&v)[N]) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float f = p.relu2 ? squared_relu(to_f(v[e])) : to_f(v[e]);
            top = max(top, __float_as_uint(f) & 0x7fffffffu);
            ss = fmaf(f, f, ss);
        }
    };
    T v[NP ? NP : 1][N];
    if constexpr (NP > 0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int at = tid + i * TPR;
            if (at < pieces) fetch(at, v[i]);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i)
            if (tid + i * TPR < pieces) look(v[i]);
    } else {
        for (int at = tid; at < pieces; at += TPR) {
            fetch(at, v[0]);
            look(v[0]);
        }
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        ss += __shfl_xor_sync(0xffffffffu, ss, off);
    }
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32;
        __shared__ unsigned s_top[W];
        __shared__ float s_ss[W];
        if ((threadIdx.x & 31) == 0) { s_top[warp] = top; s_ss[warp] = ss; }
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) { top = max(top, s_top[w]); ss += s_ss[w]; }
    }
    const bool number = top < 0x7f800000u;
    const float most = __uint_as_float(top);
    if (tid == 0) {
        float s = most;
        if (p.norm) s = most * (1.0f / sqrtf(ss * p.inv_n + p.eps));
        p.scale[row] = !number ? __uint_as_float(0x7fc00000u) : top == 0 ? 0.f : s / MOST;
    }
    const bool some = number && top != 0;
    const float r = some ? MOST / most : 0.f;
    const bool wide = !(r < __uint_as_float(0x7f800000u));
    auto put = [&](int at, const T (&v)[N]) {
        const int n = min(N, p.C - at * N);
        if (sum) store_piece<T, VEC>(sum + (long long)at * N, n, v);
        uint32_t c[N / 4];
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            float f[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = p.relu2 ? squared_relu(to_f(v[e + k])) : to_f(v[e + k]);
            c[e / 4] = some ? q8::codes_of<I8>(f, r, MOST, most, wide) : 0u;
        }
        uint8_t* to = codes + (long long)at * N;
        if (n == N) {                                            // rows of codes start on 16-byte boundaries
            if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(c[0], c[1]);
            else *reinterpret_cast<uint32_t*>(to) = c[0];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e < n) to[e] = (uint8_t)(c[e / 4] >> (8 * (e & 3)));
        }
    };
    if constexpr (NP > 0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int at = tid + i * TPR;
            if (at < pieces) put(at, v[i]);
        }
    } else {
        for (int at = tid; at < pieces; at += TPR) {
            fetch(at, v[0]);
            put(at, v[0]);
        }
    }
}

template <typename T, bool I8, bool VEC>
int quant_launch(deers_ctx* ctx, const QuantParams& p) {
    const int pieces = (p.C + Piece<T>::N - 1) / Piece<T>::N;
    KernelTimerScope ts(ctx, DEERS_K_NORM);
    const unsigned rows = (unsigned)p.rows;
    if (pieces <= 32) DEERS_CUDA_TRY(ctx, launch_chained(ctx, quantize_rows_kernel<T, I8, VEC, 32, 1>, (rows + 7) / 8, 256, 0, 1, p));
    else if (pieces <= 128) DEERS_CUDA_TRY(ctx, launch_chained(ctx, quantize_rows_kernel<T, I8, VEC, 32, 4>, (rows + 7) / 8, 256, 0, 1, p));
    else if (pieces <= 512) DEERS_CUDA_TRY(ctx, launch_chained(ctx, quantize_rows_kernel<T, I8, VEC, 128, 4>, rows, 128, 0, 1, p));
    else if (pieces <= 2048) DEERS_CUDA_TRY(ctx, launch_chained(ctx, quantize_rows_kernel<T, I8, VEC, 512, 4>, rows, 512, 0, 1, p));
    else DEERS_CUDA_TRY(ctx, launch_chained(ctx, quantize_rows_kernel<T, I8, VEC, 512, 0>, rows, 512, 0, 1, p));
    return DEERS_OK;
}

}  // namespace

extern "C" int deers_b200_quantize_rows(deers_ctx* ctx, const deers_quantize_desc* d, const void* x, const void* residual, void* sum,
                                        void* codes, float* scale) {
    if (!ctx || !d) return DEERS_ERR_NULL;
    if (d->dtype != DEERS_F16 && d->dtype != DEERS_F32) return DEERS_ERR_DTYPE;
    if (d->code != DEERS_I8 && d->code != DEERS_E4M3) return DEERS_ERR_DTYPE;
    if (d->rows < 0 || d->rows > 0x7fffffffLL || d->C < 1) return DEERS_ERR_SHAPE;
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
    p.norm = d->norm; p.relu2 = d->relu_squared;
    const bool vec = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)sum) & 15u) == 0 &&
                     ((p.ld_x | p.ld_res | p.ld_sum) * (long long)es & 15) == 0;
    const bool half = d->dtype == DEERS_F16, i8 = d->code == DEERS_I8;
    const auto go = half ? (i8 ? (vec ? quant_launch<__half, true, true> : quant_launch<__half, true, false>)
                               : (vec ? quant_launch<__half, false, true> : quant_launch<__half, false, false>))
                         : (i8 ? (vec ? quant_launch<float, true, true> : quant_launch<float, true, false>)
                               : (vec ? quant_launch<float, false, true> : quant_launch<float, false, false>));
    const int rc = go(ctx, p);
    if (rc) return rc;
    ctx->launches += 1;
    DEERS_CUDA_TRY(ctx, cudaGetLastError());
    return DEERS_OK;
}
