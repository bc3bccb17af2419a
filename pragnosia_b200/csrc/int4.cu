// Weights in four bits with a scale per group, and the linear layer that reads them.
//
//   A weight (N, K), K a multiple of 32, is q [N][K/2] bytes (the even column in the low half), and for each group of g = 32, 64 or 128 columns of a row
//   (the last may be shorter) a scale s in bf16 or fp32 and a whole number z [N][G] bytes (none: 8 everywhere). It stands for w' = s (q - z).
//
//   quantise   lo = min(0, min w), hi = max(0, max w) of the group
//              with zeros:  s = (hi - lo) / 15, z = clamp(rint(-lo / s), 0, 15);   without:  s = max|w| / 7, z = 8
//              q = clamp(rint(w / s) + z, 0, 15);   s is rounded to its type before it is used, and s = 0 gives q = z
//   linear     y = act(x W'^T + b)
//
// Every step of the quantisation is one correctly rounded fp32 operation, so the same weights give the same levels anywhere. A group that holds an
// infinity or NaN has a scale of NaN, and so has one whose range leaves fp32.
#include "tc_common.cuh"

namespace pgb {

// ------------------------------------------------------------------------------------------------ quantise, read back
// A thread owns eight columns: 16 or 32 bytes in, 4 out; the threads of a group are neighbours in a warp.
template <typename T_> __device__ __forceinline__ void load8(const T_ *p, float (&f)[8]) {
    if constexpr (sizeof(T_) == 2) {
        const uint4 r = *reinterpret_cast<const uint4 *>(p);
        const __nv_bfloat162 *b = reinterpret_cast<const __nv_bfloat162 *>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 t = __bfloat1622float2(b[i]); f[2 * i] = t.x; f[2 * i + 1] = t.y; }
    } else {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
}
template <typename T_> __device__ __forceinline__ void store8(T_ *p, const float (&f)[8]) {
    if constexpr (sizeof(T_) == 2) {
        uint4 r;
        __nv_bfloat162 *b = reinterpret_cast<__nv_bfloat162 *>(&r);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = r;
    } else {
        reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
}

template <typename T_, int GROUP>
__global__ void __launch_bounds__(256) int4_quantize_kernel(const T_ *__restrict__ w, unsigned char *__restrict__ q, T_ *__restrict__ scales,
                                                            unsigned char *__restrict__ zeros, int N, int K, int G) {
    constexpr int PER = GROUP / 8;                                    // threads of a group
    const long long idx = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long grp = idx / PER;                                  // row-major over (N, G)
    const int part = (int)(idx % PER);
    const bool row_live = grp < (long long)N * G;
    const int n = row_live ? (int)(grp / G) : 0, col = row_live ? (int)(grp % G) * GROUP + part * 8 : K;
    const bool live = row_live && col < K;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};            // zeros change no group's range
    if (live) load8(w + (size_t)n * K + col, f);
    float lo = 0.f, hi = 0.f, bad = 0.f;                              // bad: NaN where a value is not finite (x - x), else 0
#pragma unroll
    for (int i = 0; i < 8; ++i) { lo = fminf(lo, f[i]); hi = fmaxf(hi, f[i]); bad += f[i] - f[i]; }
#pragma unroll
    for (int o = PER / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        bad += __shfl_xor_sync(0xffffffffu, bad, o);
    }
    const bool sym = zeros == nullptr;
    T_ st;
    from_f32(st, sym ? __fdiv_rn(fmaxf(-lo, hi), 7.f) : __fdiv_rn(__fsub_rn(hi, lo), 15.f));
    float s = to_f32(st);
    if (bad != 0.f || !(s < INFINITY)) { s = nanf(""); from_f32(st, s); }
    const bool flat = !(s > 0.f);                                     // no range, or NaN
    const float z = sym ? 8.f : flat ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f);
    if (!live) return;
    uint32_t packed = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = flat ? z : fminf(fmaxf(rintf(__fdiv_rn(f[i], s)) + z, 0.f), 15.f);
        packed |= (uint32_t)r << (4 * i);
    }
    *reinterpret_cast<uint32_t *>(q + ((size_t)n * K + col) / 2) = packed;
    if (part == 0) {
        scales[grp] = st;
        if (!sym) zeros[grp] = (unsigned char)z;
    }
}

template <typename T_, typename O_>
__global__ void __launch_bounds__(256) int4_dequantize_kernel(const unsigned char *__restrict__ q, const T_ *__restrict__ scales,
                                                              const unsigned char *__restrict__ zeros, O_ *__restrict__ w, int N, int K, int G, int lg) {
    const long long i8 = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i8 >= (long long)N * K / 8) return;
    const int per = K / 8, n = (int)(i8 / per), col = (int)(i8 % per) * 8;
    const size_t at = (size_t)n * G + (col >> lg);
    const uint32_t p = reinterpret_cast<const uint32_t *>(q)[i8];
    const float s = to_f32(scales[at]), z = zeros != nullptr ? (float)zeros[at] : 8.f;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = s * ((float)((p >> (4 * i)) & 15u) - z);
    store8(w + (size_t)i8 * 8, f);
}

// ------------------------------------------------------------------------------------------------ linear
__device__ __forceinline__ float int4_act(float v, int act) { return act == 1 ? 0.5f * v * (1.0f + erff(v * 0.70710678118654752f)) : v; }

// Tiles of 64 x 64 in fp32, a group's sum of whole numbers times x scaled once.
template <typename X_, typename S_, typename O_>
__global__ void __launch_bounds__(256) int4_linear_tile_kernel(const X_ *__restrict__ x, const unsigned char *__restrict__ q, const S_ *__restrict__ scales,
                                                               const unsigned char *__restrict__ zeros, const X_ *__restrict__ bias, int act,
                                                               O_ *__restrict__ y, long long M, int N, int K, int G, int lg) {
    __shared__ float xs[32][65], ws[32][65];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int n0 = blockIdx.x * 64;
    const long long m0 = (long long)blockIdx.y * 64;
    float acc[4][4] = {}, part[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 32) {
        const int r = tid >> 2, c = (tid & 3) * 8;
        float f[8] = {};
        if (m0 + r < M) load8(x + (size_t)(m0 + r) * K + k0 + c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) xs[c + i][r] = f[i];
        uint32_t p = 0;
        float z = 8.f;
        if (n0 + r < N) {
            p = *reinterpret_cast<const uint32_t *>(q + ((size_t)(n0 + r) * K + k0 + c) / 2);
            if (zeros != nullptr) z = (float)zeros[(size_t)(n0 + r) * G + (k0 >> lg)];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ws[c + i][r] = (float)((p >> (4 * i)) & 15u) - z;
        __syncthreads();
#pragma unroll 8
        for (int k = 0; k < 32; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(xs[k][ty + 16 * i], ws[k][tx + 16 * j], part[i][j]);
        __syncthreads();
        if (k0 + 32 >= K || ((k0 + 32) >> lg) != (k0 >> lg)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int n = n0 + tx + 16 * j;
                const float s = n < N ? to_f32(scales[(size_t)n * G + (k0 >> lg)]) : 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) { acc[i][j] = fmaf(s, part[i][j], acc[i][j]); part[i][j] = 0.f; }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + ty + 16 * i;
            const int n = n0 + tx + 16 * j;
            if (m < M && n < N) from_f32(y[(size_t)m * N + n], int4_act(acc[i][j] + (bias != nullptr ? to_f32(bias[n]) : 0.f), act));
        }
}

// ------------------------------------------------------------------------------------------------ host
static inline int log2_group(int group) { return group == 32 ? 5 : group == 64 ? 6 : 7; }

template <typename T_>
static void quantize_go(const void *w, unsigned char *q, void *scales, unsigned char *zeros, int N, int K, int group, cudaStream_t stream) {
    const int G = (K + group - 1) / group;
    const unsigned grid = (unsigned)(((long long)N * G * (group / 8) + 255) / 256);
    const T_ *wp = (const T_ *)w;
    T_ *sp = (T_ *)scales;
    if (group == 32) int4_quantize_kernel<T_, 32><<<grid, 256, 0, stream>>>(wp, q, sp, zeros, N, K, G);
    else if (group == 64) int4_quantize_kernel<T_, 64><<<grid, 256, 0, stream>>>(wp, q, sp, zeros, N, K, G);
    else int4_quantize_kernel<T_, 128><<<grid, 256, 0, stream>>>(wp, q, sp, zeros, N, K, G);
}
int int4_quantize_launch(const void *w, int dtype, unsigned char *q, void *scales, unsigned char *zeros, int N, int K, int group, cudaStream_t stream) {
    if (dtype == PGB_BF16) quantize_go<__nv_bfloat16>(w, q, scales, zeros, N, K, group, stream);
    else quantize_go<float>(w, q, scales, zeros, N, K, group, stream);
    return check_launch("int4_quantize_kernel");
}

int int4_dequantize_launch(const Int4Weight &w, void *out, int out_dtype, cudaStream_t stream) {
    const unsigned grid = (unsigned)(((long long)w.N * w.K / 8 + 255) / 256);
    const int lg = log2_group(w.group);
    const bool sb = w.scale_dtype == PGB_BF16, ob = out_dtype == PGB_BF16;
    const __nv_bfloat16 *s16 = (const __nv_bfloat16 *)w.scales;
    const float *s32 = (const float *)w.scales;
    if (sb && ob) int4_dequantize_kernel<<<grid, 256, 0, stream>>>(w.q, s16, w.zeros, (__nv_bfloat16 *)out, w.N, w.K, w.G, lg);
    else if (sb) int4_dequantize_kernel<<<grid, 256, 0, stream>>>(w.q, s16, w.zeros, (float *)out, w.N, w.K, w.G, lg);
    else if (ob) int4_dequantize_kernel<<<grid, 256, 0, stream>>>(w.q, s32, w.zeros, (__nv_bfloat16 *)out, w.N, w.K, w.G, lg);
    else int4_dequantize_kernel<<<grid, 256, 0, stream>>>(w.q, s32, w.zeros, (float *)out, w.N, w.K, w.G, lg);
    return check_launch("int4_dequantize_kernel");
}

template <typename X_, typename S_, typename O_>
static void tile_go(const Int4Linear &a, cudaStream_t stream) {
    const Int4Weight &w = a.w;
    for (long long m = 0; m < a.M; m += 65535LL * 64) {               // a grid's second axis ends at 65535
        const long long rows = a.M - m < 65535LL * 64 ? a.M - m : 65535LL * 64;
        int4_linear_tile_kernel<<<dim3((unsigned)((w.N + 63) / 64), (unsigned)((rows + 63) / 64)), 256, 0, stream>>>(
            (const X_ *)a.x + (size_t)m * w.K, w.q, (const S_ *)w.scales, w.zeros, (const X_ *)a.bias, a.act, (O_ *)a.y + (size_t)m * w.N, rows, w.N, w.K, w.G,
            log2_group(w.group));
    }
}
template <typename X_>
static void tile_types(const Int4Linear &a, cudaStream_t stream) {
    const bool sb = a.w.scale_dtype == PGB_BF16, ob = a.out_dtype == PGB_BF16;
    if (sb && ob) tile_go<X_, __nv_bfloat16, __nv_bfloat16>(a, stream);
    else if (sb) tile_go<X_, __nv_bfloat16, float>(a, stream);
    else if (ob) tile_go<X_, float, __nv_bfloat16>(a, stream);
    else tile_go<X_, float, float>(a, stream);
}
int int4_linear_launch(const Int4Linear &a, cudaStream_t stream) {
    if (a.x_dtype == PGB_BF16) tile_types<__nv_bfloat16>(a, stream);
    else tile_types<float>(a, stream);
    return check_launch("int4_linear_tile_kernel");
}

}  // namespace pgb
