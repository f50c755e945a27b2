// New keys and values into a cache of e4m3 codes with a scale for every 32 tokens of a head.
//
// Row start[b] + t of sequence b receives new row t, t < count[b].  Of a block of 32 tokens that gets rows,
//     scale' = max(scale if the block holds earlier rows of the sequence, max|new rows| * (1 / 448 in f32))
// new codes are nearest(value / scale'), and where the scale has grown the block's earlier rows are rounded again, nearest(code * scale / scale');
// other rows and blocks stay as they are.  So one scale serves a block however its rows arrive, a block that starts anew forgets what lay
// there, and writing the same rows again changes nothing.  A value that is no number is stored as NaN and takes no part in the scale.
// A group of threads (a warp, or four) owns a block of one head of keys or values: it reads the new rows once, into registers.
// Bound: HBM, 3 bytes an element with f16 (8 x 8 heads of 2048 rows of 256 33.8 us, 5.2 TB/s; f32 46.4, 6.3), instructions below 256 channels (of 128 20.0 us,
// 4.4 TB/s; f32 24.3, 6.0); for single tokens the launch.  Values next to a border between codes are decided last: f16 24 -> 21 us, f32 27 -> 24.
#include "common.cuh"
#include "q8_codes.cuh"

namespace {

struct AppendParams {
    const void* src[2];                       // keys, values [B,H,T,D]
    uint8_t* codes[2];                        // [B,H,cap,D]
    float* scale[2];                          // [B,H,blocks]
    long long ss[2][3], sc[2][3], sl[2][2];   // strides (b, h, t) in elements, of the scales (b, h)
    const int* start; const int* count;       // count may be nullptr: T rows of every sequence
    int H, T, D, cap;
    unsigned int* told;
};

__device__ __forceinline__ float as_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_f(float v) { return v; }
__device__ __forceinline__ __half not_a_number(__half) { return __ushort_as_half(0x7e00); }
__device__ __forceinline__ float not_a_number(float) { return __uint_as_float(0x7fc00000u); }

// 32 * NW threads own a token block, LR threads a row of it, eight values each; NP rows of a thread stay in registers.  Whole blocks of f16 hide
// their loads behind other blocks: ten on an SM for heads up to 64 (14.2 -> 13.2 us for 8 x 8 heads of 2048 rows), eight up to 128 (20.7 -> 20.0);
// wider ones have 64 values a thread, and are quicker with the registers that they ask for (39.3 -> 33.8).
template <typename T, bool VEC, int LR, int NW, int NP>
__global__ void __launch_bounds__(128, NW == 4 && sizeof(T) == 2 ? (LR == 8 ? 10 : LR == 16 ? 8 : 1) : 1) append_q8_kernel(const AppendParams p) {
    chain_begin();
    constexpr int NT = 32 * NW, PER = 128 / NT, STEP = NT / LR;  // groups of a block of threads; rows at a time
    const int tid = threadIdx.x % NT, warp = threadIdx.x / 32;
    const int h = blockIdx.y * PER + threadIdx.x / NT, b = blockIdx.z >> 1, kv = blockIdx.z & 1;
    const bool mine = h < p.H;                                   // (with NW == 4 the whole block)
    int begin = p.start[b], n = p.count ? p.count[b] : p.T;
    if (n < 0 || n > p.T || (n > 0 && (begin < 0 || (long long)begin + n > p.cap))) {      // rows outside of the cache are left out, and told
        if (threadIdx.x == 0 && blockIdx.x == 0) atomicCAS(p.told, 0u, (unsigned)DEERS_KERR_CACHE | 1u);
        n = min(max(n, 0), p.T);
        if (begin < 0 || begin >= p.cap) n = 0;
        n = min(n, p.cap - begin);
    }
    if (n <= 0 || !mine) return;
    const int blk = begin / q8::BLOCK + blockIdx.x, first = blk * q8::BLOCK;
    const int lo = max(begin, first), hi = min(begin + n, first + q8::BLOCK);
    if (lo >= hi) return;
    uint8_t* codes = p.codes[kv] + b * p.sc[kv][0] + h * p.sc[kv][1];
    float* scale_at = p.scale[kv] + b * p.sl[kv][0] + h * p.sl[kv][1] + blk;
    const int row = tid / LR, col = tid % LR * 8, rows = col < p.D ? hi - lo - row : 0;      // this thread's: row, row + STEP, ..
    const T* src = static_cast<const T*>(p.src[kv]) + b * p.ss[kv][0] + h * p.ss[kv][1] + (long long)(lo - begin + row) * p.ss[kv][2] + col;
    const float was = begin > first ? *scale_at : 0.f;
    T v[NP][8];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        if (i * STEP < rows) {
            const T* s = src + i * STEP * p.ss[kv][2];
            if constexpr (VEC) {
#pragma unroll
                for (int w = 0; w < (int)sizeof(T) / 2; ++w) reinterpret_cast<uint4*>(v[i])[w] = reinterpret_cast<const uint4*>(s)[w];
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = s[e];
            }
        }
    }
    auto most = [&]() {                                          // the group's largest |value|, NaN passed over
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (i * STEP < rows) q8::look_at8(top, v[i]);
        }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        if constexpr (NW > 1) {
            __shared__ float s_top[4];
            __syncthreads();
            if ((threadIdx.x & 31) == 0) s_top[warp] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) top = fmaxf(top, s_top[w]);
        } else {
            __syncwarp();                                        // every lane has read the old scale
        }
        return top;
    };
    const float inf = __uint_as_float(0x7f800000u);
    float top = most();
    if (!(top < inf)) {                                          // infinities are no part of the scale, and are stored as NaN
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (fabsf(as_f(v[i][e])) == inf) v[i][e] = not_a_number(v[i][e]);
        top = most();
    }
    const float fresh = top * (1.0f / q8::MOST_E4M3);
    const bool grown = fresh > was;
    const float scale = grown ? fresh : was;
    if (tid == 0) *scale_at = scale;
    const float den = scale > 0.f ? scale : 1.0f;
    const q8::Factors factors = q8::factors(1.0f, den, q8::den_is_far(den));
    uint8_t* to = codes + (lo + row) * p.sc[kv][2] + col;
    uint32_t near = 0;                                           // groups of four values that hold one next to a border
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        if (i * STEP < rows) {
            uint32_t c[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float f[4];
                uint32_t up;
                q8::four(v[i] + 4 * k, f);
                q8::bounds_e4m3(f, factors, c[k], up);
                if (c[k] != up) near |= 1u << (2 * i + k);
            }
            *reinterpret_cast<uint2*>(to + i * STEP * p.sc[kv][2]) = make_uint2(c[0], c[1]);
        }
    }
    // They are decided behind everything else, from memory again: a call where the rows' registers live costs more than its own time.
#pragma unroll 1
    for (; near; near &= near - 1) {
        const int j = __ffs((int)near) - 1, i = j >> 1, k = j & 1;
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = as_f(src[i * STEP * p.ss[kv][2] + 4 * k + e]);
            if (fabsf(f[e]) == inf) f[e] = __uint_as_float(0x7fc00000u);
        }
        *reinterpret_cast<uint32_t*>(to + i * STEP * p.sc[kv][2] + 4 * k) = q8::quotients_e4m3(f[0], f[1], f[2], f[3], 1.0f, den);
    }
    if (grown && begin > first) {                                // the earlier rows, 16 bytes at a time
        const q8::Factors again = q8::factors(was, scale, q8::den_is_far(scale) || !(was > 1e-20f));
        const int per16 = p.D / 16, old16 = (begin - first) * per16;
        for (int at = tid; at < old16; at += NT) {
            uint4* c = reinterpret_cast<uint4*>(codes + (first + at / per16) * p.sc[kv][2] + at % per16 * 16);
            const uint4 w = *c;
            const uint32_t in[4] = {w.x, w.y, w.z, w.w};
            uint32_t out[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[4];
                q8::e4m3_values(in[k], f);
                out[k] = q8::codes_of<false>(f, again, was, scale);
            }
            *c = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
}

// A warp for a token block that gets few rows, four warps otherwise.
template <typename T, bool VEC, int LR>
int append_widths(deers_ctx* ctx, const AppendParams& p, int B) {
    // token blocks that T rows can touch from any place
    const unsigned blocks = p.T < 2 ? 1u : (unsigned)((p.T - 2) / q8::BLOCK + 2);
    KernelTimerScope ts(ctx, DEERS_K_DECODE);
    const dim3 warps(blocks, (unsigned)((p.H + 3) / 4), 2u * B), whole(blocks, (unsigned)p.H, 2u * B);
    if (p.T <= 32 / LR) DEERS_CUDA_TRY(ctx, launch_chained(ctx, append_q8_kernel<T, VEC, LR, 1, 1>, warps, 128, 0, 1, p));
    else if (p.T <= 128 / LR) DEERS_CUDA_TRY(ctx, launch_chained(ctx, append_q8_kernel<T, VEC, LR, 1, 4>, warps, 128, 0, 1, p));
    else DEERS_CUDA_TRY(ctx, launch_chained(ctx, append_q8_kernel<T, VEC, LR, 4, LR / 4>, whole, 128, 0, 1, p));
    return DEERS_OK;
}
template <typename T, bool VEC>
int append_launch(deers_ctx* ctx, const AppendParams& p, int B) {
    return p.D <= 64 ? append_widths<T, VEC, 8>(ctx, p, B) : p.D <= 128 ? append_widths<T, VEC, 16>(ctx, p, B) : append_widths<T, VEC, 32>(ctx, p, B);
}

}  // namespace

int deers_check_cache(const deers_cache_q8* c) {
    if (!c) return DEERS_ERR_NULL;
    if (c->B < 1 || c->H < 1 || c->capacity < 1 || c->D < 1) return DEERS_ERR_SHAPE;
    if (c->D % 16 || c->D > 256 || c->B > 32767 || c->H > 65535 || c->capacity > (1 << 24) || c->k_strides[2] > (1 << 26) || c->v_strides[2] > (1 << 26))
        return DEERS_ERR_UNSUPPORTED;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return DEERS_ERR_NULL;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u || ((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3u) return DEERS_ERR_LAYOUT;
    for (int i = 0; i < 3; ++i)
        if (c->k_strides[i] < 0 || c->v_strides[i] < 0 || (c->k_strides[i] | c->v_strides[i]) & 15) return DEERS_ERR_LAYOUT;
    for (int i = 0; i < 2; ++i)
        if (c->k_scale_strides[i] < 0 || c->v_scale_strides[i] < 0) return DEERS_ERR_LAYOUT;
    if (c->k_strides[2] < c->D || c->v_strides[2] < c->D) return DEERS_ERR_LAYOUT;
    return DEERS_OK;
}

extern "C" int deers_b200_cache_q8_append(deers_ctx* ctx, const deers_cache_q8* c, int32_t T, int32_t dtype, const void* k, const int64_t* k_strides,
                                          const void* v, const int64_t* v_strides, const int32_t* start, const int32_t* count) {
    if (!ctx || !c || !k_strides || !v_strides) return DEERS_ERR_NULL;
    int rc = deers_check_cache(c);
    if (rc) return rc;
    if (dtype != DEERS_F16 && dtype != DEERS_F32) return DEERS_ERR_DTYPE;
    if (T < 0 || T > c->capacity) return DEERS_ERR_SHAPE;
    if (T == 0) return DEERS_OK;
    if (!k || !v || !start) return DEERS_ERR_NULL;
    const int64_t es = dtype == DEERS_F16 ? 2 : 4;
    if (((uintptr_t)k | (uintptr_t)v) & (uintptr_t)(es - 1) || ((uintptr_t)start | (uintptr_t)count) & 3u) return DEERS_ERR_LAYOUT;
    if (k_strides[3] != 1 || v_strides[3] != 1) return DEERS_ERR_LAYOUT;
    bool vec = (((uintptr_t)k | (uintptr_t)v) & 15u) == 0;
    AppendParams p;
    for (int i = 0; i < 3; ++i) {
        if (k_strides[i] < 0 || v_strides[i] < 0) return DEERS_ERR_LAYOUT;
        // (a cache whose sequences or heads are one place can be read, not written)
        if ((i == 0 ? c->B : i == 1 ? c->H : 1) > 1 && (c->k_strides[i] == 0 || c->v_strides[i] == 0)) return DEERS_ERR_LAYOUT;
        vec = vec && ((k_strides[i] | v_strides[i]) * es & 15) == 0;
        p.ss[0][i] = k_strides[i]; p.ss[1][i] = v_strides[i];
        p.sc[0][i] = c->k_strides[i]; p.sc[1][i] = c->v_strides[i];
    }
    for (int i = 0; i < 2; ++i)
        if ((i == 0 ? c->B : c->H) > 1 && (c->k_scale_strides[i] == 0 || c->v_scale_strides[i] == 0)) return DEERS_ERR_LAYOUT;
    for (int i = 0; i < 2; ++i) { p.sl[0][i] = c->k_scale_strides[i]; p.sl[1][i] = c->v_scale_strides[i]; }
    p.src[0] = k; p.src[1] = v;
    p.codes[0] = (uint8_t*)c->k; p.codes[1] = (uint8_t*)c->v;
    p.scale[0] = c->k_scale; p.scale[1] = c->v_scale;
    p.start = start; p.count = count;
    p.H = c->H; p.T = T; p.D = c->D; p.cap = c->capacity; p.told = ctx->dev_err + 1;
    DEERS_CUDA_TRY(ctx, cudaSetDevice(ctx->device));
    const auto go = dtype == DEERS_F16 ? (vec ? append_launch<__half, true> : append_launch<__half, false>)
                                       : (vec ? append_launch<float, true> : append_launch<float, false>);
    if ((rc = go(ctx, p, c->B))) return rc;
    ctx->launches += 1;
    DEERS_CUDA_TRY(ctx, cudaGetLastError());
    return DEERS_OK;
}
