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

// Few rows of x: the time is the weight's bytes, and what stands in their way is the arithmetic that makes operands of them. One CTA owns 16 MT rows of W, its
// eight warps every eighth stretch of 128 columns each. A warp streams its stretches through slots of shared memory of its own by asynchronous copies (nothing
// is held in registers while they fly, no barrier between warps), so a CTA reads 512 B of each row at a time, and the warps' sums meet once at the end, in order.
//   Operands of the warp-level m16n8k16 product: the whole numbers q - z in bf16 (exact: 0x4300 | q is 128 + q, less 128 + z), 16 rows of W by 16 columns, and up to
// 8 rows of x. A word of eight levels k0..k7 gives pairs (k0,k4), (k1,k5), (k2,k6), (k3,k7) with a shift and a mask each, so the product's 16 columns are taken in
// that order and x, whose fragments serve all MT blocks of rows, is reordered by byte permutes. A group's products end in an accumulator of their own that enters the
// sum times the scale: the weight is never rounded. fp32 rows of x are three terms of eight bits each, cut off (their sum is x to the last bit), three products.
//   Levels lie in 64-byte rows whose 16-byte pieces are swapped by the row, so that the eight rows of a fragment's word touch every bank once.
constexpr int RW_WARPS = 8, RW_NT = RW_WARPS * 32;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes) {      // bytes 0: zeros
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N_> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N_) : "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma_bf16_warp(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the pair of levels in bits 0-3 and 16-19 as bf16 whole numbers less the zero: z2 is 128 + z twice
__device__ __forceinline__ uint32_t level_pair(uint32_t w, uint32_t z2) {
    uint32_t v = (w & 0x000f000fu) | 0x43004300u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&v), *reinterpret_cast<const __nv_bfloat162 *>(&z2));
    return *reinterpret_cast<const uint32_t *>(&d);
}

struct RowsArgs {
    const void *x; const unsigned char *q; const void *scales; const unsigned char *zeros; const void *bias; void *y;
    int act, out_bf16, N, K, G, lg, slots, slot_bytes, constant;
    long long M;
};

template <int MT, int NB, bool X32, bool S32>
__global__ void __launch_bounds__(RW_NT) int4_rows_kernel(const RowsArgs a) {
    constexpr int R = 16 * MT, RP = R + 4, TERMS = X32 ? 3 : 1;
    extern __shared__ __align__(1024) uint8_t rw_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * R, rows = a.M - (long long)blockIdx.y * (8 * NB) < 8 * NB ? (int)(a.M - (long long)blockIdx.y * (8 * NB)) : 8 * NB;
    const long long m0 = (long long)blockIdx.y * (8 * NB);
    const int C = (a.K + 127) >> 7, mine = C > warp ? (C - warp + RW_WARPS - 1) / RW_WARPS : 0;     // stretches, and this warp's
    const uint32_t ring = smem_u32(rw_smem) + warp * a.slots * a.slot_bytes;
    const uint8_t *xg = reinterpret_cast<const uint8_t *>(a.x) + m0 * a.K * (X32 ? 4 : 2);

    auto fetch_w = [&](int i) {                                       // stretch i of this warp into its slot
        const int k = (warp + i * RW_WARPS) * 128 + (lane & 3) * 32;
        const uint32_t dst = ring + (i % a.slots) * a.slot_bytes;
#pragma unroll
        for (int u = 0; u < 2 * MT; ++u) {
            const int r = u * 8 + (lane >> 2);
            const bool in = n0 + r < a.N && k < a.K;
            cp_async16(dst + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4), a.q + (in ? ((size_t)(n0 + r) * a.K + k) / 2 : 0), in ? 16 : 0);
        }
    };
    // x: pieces of 64 B (32 columns of bf16, 16 of fp32), [piece][row]
    auto fetch_x = [&](int i) {
        const uint32_t dst = ring + (i % a.slots) * a.slot_bytes + R * 64;
        constexpr int PIECES = X32 ? 8 : 4, E = X32 ? 4 : 2;
        const int c0 = (warp + i * RW_WARPS) * 128;
        for (int u = lane; u < PIECES * rows * 4; u += 32) {
            const int c = u & 3, pr = u >> 2, p = pr / rows, r = pr - p * rows;
            const int k = c0 + (p * 64 + c * 16) / E;
            const bool in = k < a.K;
            cp_async16(dst + u * 16, xg + (in ? ((size_t)r * a.K + k) * E : 0), in ? 16 : 0);
        }
    };
    // scales and zeros of this lane's rows, group t of the stretch: the scale's bits, or (bf16) those and 128 + z in one word
    uint32_t sc[2][MT], zr[2][S32 ? MT : 1];
    auto fetch_s = [&](int i) {
        const int grp = (((warp + i * RW_WARPS) * 128) >> a.lg) + t;
        const bool in = i < mine && t < (128 >> a.lg) && grp < a.G;
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + 16 * u + 8 * h + g;
                const size_t at = (size_t)(n < a.N ? n : a.N - 1) * a.G + grp;
                const uint32_t z = 0x4300u | (in && a.zeros != nullptr ? a.zeros[at] : 8u);
                if constexpr (S32) {
                    sc[h][u] = in ? reinterpret_cast<const uint32_t *>(a.scales)[at] : 0u;
                    zr[h][u] = z;
                } else {
                    sc[h][u] = (in ? (uint32_t)reinterpret_cast<const unsigned short *>(a.scales)[at] << 16 : 0u) | z;
                }
            }
    };

    if (!a.constant) { pdl_wait(); pdl_launch_dependents(); }
    const int ahead = a.slots - 1;
    if (a.constant) {
        for (int i = 0; i < ahead && i < mine; ++i) fetch_w(i);
        fetch_s(0);
        pdl_launch_dependents();
        pdl_wait();
        for (int i = 0; i < ahead && i < mine; ++i) fetch_x(i);
        cp_async_commit();                                            // one group for all of them; the empty ones keep the count
        for (int i = 1; i < ahead; ++i) cp_async_commit();
    } else {
        for (int i = 0; i < ahead; ++i) {
            if (i < mine) { fetch_w(i); fetch_x(i); }
            cp_async_commit();
        }
        fetch_s(0);
    }

    float acc[MT][NB][4] = {}, part[MT][NB][4] = {};
    const int per = a.lg - 5;                                         // log2 of the 32-column pieces a group has
    for (int i = 0; i < mine; ++i) {
        uint32_t s0[2][MT], z0[2][S32 ? MT : 1];
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s0[h][u] = sc[h][u];
                if constexpr (S32) z0[h][u] = zr[h][u];
            }
        if (i + ahead < mine) { fetch_w(i + ahead); fetch_x(i + ahead); }
        cp_async_commit();
        fetch_s(i + 1);
        if (a.slots == 2) cp_async_wait<1>(); else if (a.slots == 3) cp_async_wait<2>(); else if (a.slots == 4) cp_async_wait<3>();
        else if (a.slots == 5) cp_async_wait<4>(); else cp_async_wait<5>();
        __syncwarp();
        const uint32_t ws = ring + (i % a.slots) * a.slot_bytes, xs = ws + R * 64;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // x: columns 32 j + 8 t .. + 7 of row 8 b + g, as (0,4) (1,5) (2,6) (3,7)
            uint32_t bx[TERMS][NB][4];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int r = 8 * b + g;
                if constexpr (!X32) {
                    uint4 v = make_uint4(0u, 0u, 0u, 0u);
                    if (r < rows) v = lds128(xs + (j * rows + r) * 64 + t * 16);
                    bx[0][b][0] = __byte_perm(v.x, v.z, 0x5410); bx[0][b][1] = __byte_perm(v.x, v.z, 0x7632);
                    bx[0][b][2] = __byte_perm(v.y, v.w, 0x5410); bx[0][b][3] = __byte_perm(v.y, v.w, 0x7632);
                } else {
                    uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
                    if (r < rows) {
                        const uint32_t at = xs + ((2 * j + (t >> 1)) * rows + r) * 64 + (t & 1) * 32;
                        lo = lds128(at); hi = lds128(at + 16);
                    }
                    const uint32_t first[4] = {lo.x, lo.y, lo.z, lo.w}, second[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t u[2][3];
#pragma unroll
                        for (int p = 0; p < 2; ++p) {                 // x = head + middle + rest, eight bits each
                            const uint32_t bits = p == 0 ? first[e] : second[e];
                            const bool fin = (bits & 0x7f800000u) != 0x7f800000u;
                            const float f = __uint_as_float(bits);
                            const float r1 = fin ? f - __uint_as_float(bits & 0xffff0000u) : 0.f;
                            const float r2 = r1 - __uint_as_float(__float_as_uint(r1) & 0xffff0000u);
                            u[p][0] = fin ? bits : (bits & 0x007fffffu) != 0u ? 0x7fc00000u : bits;
                            u[p][1] = __float_as_uint(r1); u[p][2] = __float_as_uint(r2);
                        }
#pragma unroll
                        for (int q3 = 0; q3 < 3; ++q3) bx[q3][b][e] = __byte_perm(u[0][q3], u[1][q3], 0x7632);
                    }
                }
            }
            const int src = (lane & ~3) + (j >> per);
#pragma unroll
            for (int u = 0; u < MT; ++u) {
                const int r = 16 * u + g;
                const uint32_t wa = lds32(ws + r * 64 + ((j ^ ((r >> 1) & 3)) << 4) + 4 * t), wb = lds32(ws + (r + 8) * 64 + ((j ^ (((r + 8) >> 1) & 3)) << 4) + 4 * t);
                const uint32_t sa = __shfl_sync(0xffffffffu, s0[0][u], src), sb = __shfl_sync(0xffffffffu, s0[1][u], src);
                uint32_t za, zb;
                if constexpr (S32) { za = __shfl_sync(0xffffffffu, z0[0][u], src); zb = __shfl_sync(0xffffffffu, z0[1][u], src); }
                else { za = sa; zb = sb; }
                za = __byte_perm(za, za, 0x1010); zb = __byte_perm(zb, zb, 0x1010);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a0 = level_pair(wa >> (8 * h), za), a1 = level_pair(wb >> (8 * h), zb), a2 = level_pair(wa >> (8 * h + 4), za),
                                   a3 = level_pair(wb >> (8 * h + 4), zb);
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int q3 = TERMS - 1; q3 >= 0; --q3) mma_bf16_warp(part[u][b], a0, a1, a2, a3, bx[q3][b][2 * h], bx[q3][b][2 * h + 1]);
                }
                if (((j + 1) & ((1 << per) - 1)) == 0) {              // the group ends here
                    const float fa = __uint_as_float(S32 ? sa : sa & 0xffff0000u), fb = __uint_as_float(S32 ? sb : sb & 0xffff0000u);
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        acc[u][b][0] = fmaf(fa, part[u][b][0], acc[u][b][0]); acc[u][b][1] = fmaf(fa, part[u][b][1], acc[u][b][1]);
                        acc[u][b][2] = fmaf(fb, part[u][b][2], acc[u][b][2]); acc[u][b][3] = fmaf(fb, part[u][b][3], acc[u][b][3]);
                        part[u][b][0] = part[u][b][1] = part[u][b][2] = part[u][b][3] = 0.f;
                    }
                }
            }
        }
        __syncwarp();                                                 // the slot is read: the next copy may take it
    }
    cp_async_wait<0>();
    if (a.constant) pdl_wait();
    __syncthreads();                                                  // the slots become the sums' meeting place
    float *red = reinterpret_cast<float *>(rw_smem);                  // [warp][row of x][row of W]
    const int busy = C < RW_WARPS ? C : RW_WARPS;
    if (warp < busy) {
#pragma unroll
        for (int u = 0; u < MT; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float *p = red + (warp * 8 * NB + 8 * b + 2 * t) * RP + 16 * u + g;
                p[0] = acc[u][b][0]; p[RP] = acc[u][b][1]; p[8] = acc[u][b][2]; p[RP + 8] = acc[u][b][3];
            }
    }
    __syncthreads();
    for (int i = tid; i < R * rows; i += RW_NT) {
        const int n = i % R, m = i / R;
        if (n0 + n >= a.N) continue;
        float s = 0.f;
        for (int w = 0; w < busy; ++w) s += red[(w * 8 * NB + m) * RP + n];
        if (a.bias != nullptr) s += X32 ? reinterpret_cast<const float *>(a.bias)[n0 + n] : __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(a.bias)[n0 + n]);
        s = int4_act(s, a.act);
        const size_t at = (size_t)(m0 + m) * a.N + n0 + n;
        if (a.out_bf16) reinterpret_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(s);
        else reinterpret_cast<float *>(a.y)[at] = s;
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

template <int MT, int NB, bool X32, bool S32>
static cudaError_t rows_go(RowsArgs a, cudaStream_t stream) {
    constexpr int R = 16 * MT, RED = RW_WARPS * 8 * NB * (R + 4) * 4, MOST = 104 * 1024;     // two CTAs an SM
    const int rows = a.M < 8 * NB ? (int)a.M : 8 * NB;
    a.slot_bytes = R * 64 + rows * (X32 ? 512 : 256);
    const int mine = ((a.K + 127) / 128 + RW_WARPS - 1) / RW_WARPS;
    a.slots = MOST / (RW_WARPS * a.slot_bytes);
    if (a.slots > mine + 1) a.slots = mine + 1;
    a.slots = a.slots < 2 ? 2 : a.slots > 6 ? 6 : a.slots;
    int smem = RW_WARPS * a.slots * a.slot_bytes;
    if (smem < RED) smem = RED;
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(int4_rows_kernel<MT, NB, X32, S32>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    for (; e == cudaSuccess && a.M > 0; ) {                           // a grid's second axis ends at 65535
        const long long most = 65535LL * 8 * NB, M = a.M < most ? a.M : most, rest = a.M - M;
        a.M = M;
        e = pdl_launch(int4_rows_kernel<MT, NB, X32, S32>, dim3((unsigned)((a.N + R - 1) / R), (unsigned)((M + 8 * NB - 1) / (8 * NB))), dim3(RW_NT), (size_t)smem, stream, a);
        a.x = (const uint8_t *)a.x + (size_t)M * a.K * (X32 ? 4 : 2);
        a.y = (uint8_t *)a.y + (size_t)M * a.N * (a.out_bf16 ? 2 : 4);
        a.M = rest;
    }
    return e;
}
template <int NB, bool X32, bool S32>
static cudaError_t rows_blocks(const RowsArgs &a, cudaStream_t stream) {
    const long long tiles = (a.M + 8 * NB - 1) / (8 * NB), sms = sm_count();
    if ((a.N + 63) / 64 * tiles >= sms) return rows_go<4, NB, X32, S32>(a, stream);
    if ((a.N + 31) / 32 * tiles >= sms) return rows_go<2, NB, X32, S32>(a, stream);
    return rows_go<1, NB, X32, S32>(a, stream);
}
int int4_linear_launch(const Int4Linear &l, cudaStream_t stream) {
    const Int4Weight &w = l.w;
    const RowsArgs a{l.x, w.q, w.scales, w.zeros, l.bias, l.y, l.act, l.out_dtype == PGB_BF16, w.N, w.K, w.G, log2_group(w.group), 0, 0, l.constant, l.M};
    const bool x32 = l.x_dtype == PGB_F32, s32 = w.scale_dtype == PGB_F32;
    cudaError_t e;
    if (x32) e = s32 ? rows_blocks<1, true, true>(a, stream) : rows_blocks<1, true, false>(a, stream);
    else if (l.M <= 8) e = s32 ? rows_blocks<1, false, true>(a, stream) : rows_blocks<1, false, false>(a, stream);
    else e = s32 ? rows_blocks<2, false, true>(a, stream) : rows_blocks<2, false, false>(a, stream);
    if (e != cudaSuccess) { set_cuda_error(e, "int4_rows launch"); return PGB_ERR_CUDA; }
    return check_launch("int4_rows_kernel");
}

}  // namespace pgb
