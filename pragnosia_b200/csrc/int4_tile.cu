// The four-bit linear layer for many rows of x (bf16 in and out): y^T = W' x^T on the tensor cores.
//
//   A CTA owns 128 rows of W and NT rows of x. Its eight dequantising warps stream levels through slots of shared memory of their own by asynchronous copies,
// one row of W a lane, and write scale (q - z), rounded to bf16, to tensor memory, where it is the A operand: no trip through shared memory, and scale and zero
// are one lane's own. x comes by TMA as the B operand. D (128 lanes x NT columns of fp32) stays in tensor memory; lane = row of W, so the bias is a lane's own as well.
//   Warp w < 8 takes tensor-memory lanes 32 (w mod 4) .. and every second stretch of 128 columns; warp 8 loads x (64 columns a stage, 128-byte swizzle), warp 9 issues
// the products. Two CTAs share an SM, so one's epilogue runs under the other's products. The rounding of the weight (2^-8 of it at most) costs less than the
// result's own; kept exact, each group's products would have to be read back from tensor memory and scaled, as long as the products themselves take.
//   Few rows: the columns of W are shared out over a cluster of CTAs, whose sums meet in shared memory and are added in the order of their rank.
// Every wait is bounded; one that runs out sets the error flag and the CTA winds down.
#include "gelu.cuh"
#include "int4_linear.cuh"
#include "tc_pair.cuh"

namespace pgb {

constexpr int IT_DQ = 8, IT_NT = (IT_DQ + 2) * 32, IT_XS = 4;         // dequantising warps, threads, stages of x

struct TileArgs {
    const unsigned char *q; const void *scales; const unsigned char *zeros; const __nv_bfloat16 *bias; __nv_bfloat16 *y;
    long long M; int act, N, K, G, wide, ahead, each, splits, constant;        // wide: scales of four groups at once; ahead: stretches of levels on their way; each: a split's
};

template <int NT>
struct ItCfg {
    static constexpr int XSTAGE = NT * 128, SLOT = 32 * 64;
    static constexpr int most_ahead = NT == 128 ? 1 : NT == 64 ? 3 : 4;      // of a warp's own stretches, every second one
    static constexpr int BARS = IT_XS * XSTAGE + IT_DQ * (most_ahead + 1) * SLOT;
    static constexpr int SMEM = BARS + 256 + 1024;
    static constexpr int ROW = 128 + 4;                               // of the sums' meeting place: [row of x][row of W] fp32
    static_assert(NT * ROW * 4 <= BARS, "the sums lie where x and the levels were");
    static_assert(2 * (SMEM + 1024) <= 227 * 1024 && SMEM > 76 * 1024, "two CTAs an SM, and no third, whose tensor memory would not be there");
};

template <int NT, int LG, bool S32>
__global__ void __launch_bounds__(IT_NT, 2) int4_tile_kernel(const __grid_constant__ CUtensorMap mx, const TileArgs a) {
    using CF = ItCfg<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *sm = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t mb = base + CF::BARS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + CF::BARS + 128);
    auto x_full = [&](int s) { return mb + 8 * s; };
    auto x_empty = [&](int s) { return mb + 32 + 8 * s; };
    auto a_full = [&](int s) { return mb + 64 + 8 * s; };
    auto a_empty = [&](int s) { return mb + 80 + 8 * s; };
    const uint32_t acc_full = mb + 96, drained = mb + 104;

    const int tid = threadIdx.x, lane = tid & 31, warp = warp_uniform(tid >> 5);
    const int n0 = blockIdx.x * 128;
    const long long m0 = (long long)blockIdx.y * NT;
    const int C = (a.K + 127) >> 7, c0 = (int)blockIdx.z * a.each, mine = C - c0 < a.each ? C - c0 : a.each;     // this CTA's stretches (one at least)

    if (tid == 0) {
        for (int s = 0; s < IT_XS; ++s) { mbar_init(x_full(s), 1); mbar_init(x_empty(s), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(a_full(s), 4); mbar_init(a_empty(s), 1); }
        mbar_init(acc_full, 1);
        mbar_init(drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) tmem_alloc(smem_u32(tmem_slot), 256);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot), tA = tmem + NT;    // D: NT columns; A: two stretches of 64
    if (!a.constant) { pdl_wait(); pdl_launch_dependents(); }
    bool ok = true;

    if (warp < IT_DQ) {
        // ------------------------------------------------------------------------------------------ levels -> A
        const int sub = warp & 3, par = warp >> 2, row = n0 + 32 * sub + lane;
        const uint32_t ring = base + IT_XS * CF::XSTAGE + warp * (CF::most_ahead + 1) * CF::SLOT;
        const int half = a.K >> 1, fr = lane >> 2, ft = lane & 3, slots = a.ahead + 1;
        int wcol = (c0 + par) * 128 + ft * 32;
        const unsigned char *wsrc = a.q + (size_t)(n0 + 32 * sub + fr) * half + (wcol >> 1);
        uint32_t live = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) live |= (n0 + 32 * sub + 8 * u + fr < a.N ? 1u : 0u) << u;
        const uint32_t wdst = ring + fr * 64 + ((ft ^ ((fr >> 1) & 3)) << 4);
        auto fetch = [&](int slot) {
            const uint32_t in = wcol < a.K ? live : 0u, dst = wdst + slot * CF::SLOT;
            const unsigned char *p = wsrc;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool here = in >> u & 1u;
                cp_async16(dst + u * 512, here ? p : a.q, here ? 16 : 0);
                p += (size_t)8 * half;
            }
            wcol += 256; wsrc += 128;
        };
        // scales and zeros of the four groups that stretch i lies in; those behind the last one 0
        uint32_t sn[S32 ? 4 : 2], zn;
        auto fetch_s = [&](int i) {
            const int g0 = (((c0 + i) * 128) >> LG) & ~3;
            zn = 0x08080808u;
#pragma unroll
            for (int e = 0; e < (S32 ? 4 : 2); ++e) sn[e] = 0u;
            if (row >= a.N || i >= mine) return;
            const size_t at = (size_t)row * a.G + g0;
            if (a.wide) {
                if constexpr (S32) {
                    const uint4 v = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(a.scales) + at));
                    sn[0] = v.x; sn[1] = v.y; sn[2] = v.z; sn[3] = v.w;
                } else {
                    const uint2 v = __ldg(reinterpret_cast<const uint2 *>(reinterpret_cast<const __nv_bfloat16 *>(a.scales) + at));
                    sn[0] = v.x; sn[1] = v.y;
                }
                if (a.zeros != nullptr) zn = __ldg(reinterpret_cast<const uint32_t *>(a.zeros + at));
                return;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (g0 + e < a.G) {
                    if constexpr (S32) sn[e] = __ldg(reinterpret_cast<const uint32_t *>(a.scales) + at + e);
                    else sn[e >> 1] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short *>(a.scales) + at + e) << (16 * (e & 1));
                    if (a.zeros != nullptr) zn = (zn & ~(255u << (8 * e))) | (uint32_t)__ldg(a.zeros + at + e) << (8 * e);
                }
        };
        for (int i = 0; i < a.ahead; ++i) { if (par + 2 * i < mine) fetch(i); cp_async_commit(); }
        fetch_s(par);
        if (a.constant) { pdl_launch_dependents(); pdl_wait(); }
        const uint32_t mine_row = lane * 64, sw = (lane >> 1) & 3;
        int slot = 0;
        uint32_t round = 0;                                           // of this warp's stage: stretch i goes to stage i mod 2 = par
        for (int i = par; i < mine && ok; i += 2, ++round) {
            uint32_t sc[S32 ? 4 : 2], zc = zn;
#pragma unroll
            for (int e = 0; e < (S32 ? 4 : 2); ++e) sc[e] = sn[e];
            fetch_s(i + 2);
            if (i + 2 * a.ahead < mine) fetch(slot == 0 ? a.ahead : slot - 1);
            cp_async_commit();
            if (a.ahead == 1) cp_async_wait<1>(); else if (a.ahead == 2) cp_async_wait<2>(); else if (a.ahead == 3) cp_async_wait<3>(); else cp_async_wait<4>();
            __syncwarp();
            const uint8_t *ws = sm + (ring - base) + slot * CF::SLOT + mine_row;
            slot = slot + 1 == slots ? 0 : slot + 1;
            const uint32_t dst = tA + ((uint32_t)(32 * sub) << 16) + par * 64;
            const int first = LG == 7 ? (c0 + i) & 3 : LG == 6 ? ((c0 + i) & 1) * 2 : 0;      // of the four groups, the stretch's first
            if (round >= 1) ok = mbar_wait_warp(a_empty(par), (round + 1) & 1, 61);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < 4; ++j) {                             // 32 columns
                const int e = first + (j >> (LG - 5));
                uint32_t z2 = __byte_perm(zc, 0x43u, 0x4040 | e | e << 8), s2 = 0u;
                float sf = 0.f;
                if constexpr (S32) sf = __uint_as_float(e == 0 ? sc[0] : e == 1 ? sc[1] : e == 2 ? sc[2] : sc[3]);
                else s2 = __byte_perm(e >> 1 ? sc[1] : sc[0], 0u, e & 1 ? 0x3232 : 0x1010);
                const uint4 lv = *reinterpret_cast<const uint4 *>(ws + ((j ^ sw) << 4));
                const uint32_t wv[4] = {lv.x, lv.y, lv.z, lv.w};
                uint32_t out[16];
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    uint32_t p[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {                     // (0,4) (1,5) (2,6) (3,7)
                        p[h] = level_pair(wv[v] >> (4 * h), z2);
                        if constexpr (!S32) p[h] = mul_bf16x2(p[h], s2);
                        else {
                            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&p[h]));
                            const __nv_bfloat162 r = __floats2bfloat162_rn(f.x * sf, f.y * sf);
                            p[h] = *reinterpret_cast<const uint32_t *>(&r);
                        }
                    }
                    out[4 * v] = __byte_perm(p[0], p[1], 0x5410); out[4 * v + 1] = __byte_perm(p[2], p[3], 0x5410);
                    out[4 * v + 2] = __byte_perm(p[0], p[1], 0x7632); out[4 * v + 3] = __byte_perm(p[2], p[3], 0x7632);
                }
                tmem_st16(dst + 16 * j, out);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(a_full(par));
        }
        cp_async_wait<0>();
    } else if (warp == 8) {
        // ------------------------------------------------------------------------------------------ x
        if (a.constant) pdl_wait();
        const bool leader = elect_one();
        int it = 0;
        for (; it < 2 * mine && ok; ++it) {
            const int s = it % IT_XS;
            if (it >= IT_XS) ok = mbar_wait_warp(x_empty(s), ((it / IT_XS) + 1) & 1, 62);
            if (ok && leader) {
                mbar_expect_tx(x_full(s), CF::XSTAGE);
                tma_load_3d(base + s * CF::XSTAGE, &mx, x_full(s), c0 * 128 + it * 64, (int)m0, 0);
            }
            __syncwarp();
        }
        if (!ok)                                                      // the copies under way land before shared memory goes
            for (int k = it - 1 - IT_XS < 0 ? 0 : it - 1 - IT_XS; k < it - 1; ++k) mbar_wait_tries(x_full(k % IT_XS), (k / IT_XS) & 1);
    } else {
        // ------------------------------------------------------------------------------------------ products
        if (a.constant) pdl_wait();
        constexpr uint32_t IDESC = idesc_bf16(128, NT, 0, 0);
        int it = 0;
        for (int i = 0; i < mine && ok; ++i) {
            const int st = i & 1;
            ok = mbar_wait_warp(a_full(st), (i >> 1) & 1, 63);
            for (int kb = 0; kb < 2 && ok; ++kb, ++it) {
                const int s = it % IT_XS;
                ok = mbar_wait_warp(x_full(s), (it / IT_XS) & 1, 64);
                if (!ok) break;
                tc_fence_after();
                const uint64_t db = smem_desc(base + s * CF::XSTAGE, 16, 1024);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_bf16_ts_elect(tmem, tA + st * 64 + kb * 32 + k * 8, db + k * 2, IDESC, (it | k) != 0);
                mma_commit_elect(x_empty(s));
            }
            if (ok) mma_commit_elect(a_empty(st));
        }
        if (ok) mma_commit_elect(acc_full);
        else {                                                        // products under way end before tensor memory goes
            mma_commit_elect(drained);
            mbar_wait_tries(drained, 0);
        }
    }

    // ---------------------------------------------------------------------------------------------- epilogue
    // warp w < 8: rows 32 (w mod 4) + lane of W, rows (w / 4) NT / 2 .. of x
    if (warp < IT_DQ && ok) {
        ok = mbar_wait_warp(acc_full, 0, 65);
        tc_fence_after();
    }
    constexpr int HALF = NT / 2, STEP = HALF < 16 ? HALF : 16;
    const int sub = warp & 3, mh = (warp >> 2) * HALF;
    const uint32_t tD = tmem + ((uint32_t)(32 * sub) << 16) + mh;
    float *sums = reinterpret_cast<float *>(sm);
    if (a.splits > 1) {
        if (warp < IT_DQ && ok) {
#pragma unroll
            for (int c = 0; c < HALF; c += STEP) {
                float v[16];
                tmem_ld16_nowait(tD + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < STEP; ++e) sums[(mh + c + e) * CF::ROW + 32 * sub + lane] = v[e];
            }
        }
        cluster_sync_all();                                           // every CTA's sums are there
        const uint32_t rank = cluster_rank();
        for (int i = (int)rank * IT_NT + tid; i < 128 * NT; i += a.splits * IT_NT) {
            const int n = n0 + (i & 127), m = i >> 7;
            if (n >= a.N || m0 + m >= a.M) continue;
            float s = 0.f;
            for (int r = 0; r < a.splits; ++r) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(base + (m * CF::ROW + (i & 127)) * 4, r)));
                s += v;
            }
            if (a.bias != nullptr) s += __bfloat162float(a.bias[n]);
            a.y[(size_t)(m0 + m) * a.N + n] = __float2bfloat16_rn(a.act == 1 ? lg_gelu(s) : s);
        }
        cluster_sync_all();                                           // nobody leaves while its sums are read
    } else if (warp < IT_DQ && ok) {
        const int n = n0 + 32 * sub + lane;
        const float bias = a.bias != nullptr && n < a.N ? __bfloat162float(a.bias[n]) : 0.f;
#pragma unroll
        for (int c = 0; c < HALF; c += STEP) {
            float v[16];
            tmem_ld16_nowait(tD + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < STEP; ++e) {
                const long long m = m0 + mh + c + e;
                float s = v[e] + bias;
                if (a.act == 1) s = lg_gelu(s);
                if (m < a.M && n < a.N) a.y[(size_t)m * a.N + n] = __float2bfloat16_rn(s);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, 256);
}

template <int NT, int LG, bool S32>
static cudaError_t tile_go(const Int4Linear &l, TileArgs a, int splits, cudaStream_t stream) {
    CUtensorMap mx;
    const Int4Weight &w = l.w;
    if (!tc_make_map(&mx, l.x, 1, l.M, w.K, w.K, l.M * w.K, NT)) return cudaErrorUnknown;
    const int C = (w.K + 127) / 128;
    a.each = (C + splits - 1) / splits;
    a.splits = (C + a.each - 1) / a.each;
    const int own = (a.each + 1) / 2;
    a.ahead = own < ItCfg<NT>::most_ahead ? own : ItCfg<NT>::most_ahead;
    cudaError_t e = cudaFuncSetAttribute(int4_tile_kernel<NT, LG, S32>, cudaFuncAttributeMaxDynamicSharedMemorySize, ItCfg<NT>::SMEM);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((w.N + 127) / 128), (unsigned)((l.M + NT - 1) / NT), (unsigned)a.splits);
    cfg.blockDim = dim3(IT_NT); cfg.dynamicSmemBytes = ItCfg<NT>::SMEM; cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 1; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = (unsigned)a.splits;
    cfg.attrs = at; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, int4_tile_kernel<NT, LG, S32>, mx, a);
}
template <int NT>
static cudaError_t tile_group(const Int4Linear &l, const TileArgs &a, int splits, cudaStream_t stream) {
    const bool s32 = l.w.scale_dtype == PGB_F32;
    if (l.w.group == 32) return s32 ? tile_go<NT, 5, true>(l, a, splits, stream) : tile_go<NT, 5, false>(l, a, splits, stream);
    if (l.w.group == 64) return s32 ? tile_go<NT, 6, true>(l, a, splits, stream) : tile_go<NT, 6, false>(l, a, splits, stream);
    return s32 ? tile_go<NT, 7, true>(l, a, splits, stream) : tile_go<NT, 7, false>(l, a, splits, stream);
}

// bf16 x and y. A grid's second axis ends at 65535, so very many rows go in several launches.
int int4_tile_launch(const Int4Linear &l, cudaStream_t stream) {
    const Int4Weight &w = l.w;
    const int es = w.scale_dtype == PGB_F32 ? 4 : 2;
    TileArgs a{w.q, w.scales, w.zeros, (const __nv_bfloat16 *)l.bias, (__nv_bfloat16 *)l.y, l.M, l.act, w.N, w.K, w.G, 0, 0, 0, 1, l.constant};
    a.wide = w.G % 4 == 0 && aligned(w.scales, 4 * es) && (w.zeros == nullptr || aligned(w.zeros, 4));
    const int NT = l.M <= 32 ? 32 : l.M <= 64 ? 64 : 128, C = (w.K + 127) / 128;
    const long long tiles = (long long)((w.N + 127) / 128) * ((l.M + NT - 1) / NT);
    int splits = 1;                                                   // as many as give every SM a CTA, of two stretches or more
    while (NT < 128 && splits < 8 && tiles * splits * 2 <= sm_count() * 2 && C >= 4 * splits) splits *= 2;
    Int4Linear part = l;
    cudaError_t e = cudaSuccess;
    for (long long m = 0; m < l.M && e == cudaSuccess; m += 65535LL * NT) {
        part.M = l.M - m < 65535LL * NT ? l.M - m : 65535LL * NT;
        part.x = (const __nv_bfloat16 *)l.x + (size_t)m * w.K;
        a.M = part.M;
        a.y = (__nv_bfloat16 *)l.y + (size_t)m * w.N;
        e = NT == 32 ? tile_group<32>(part, a, splits, stream) : NT == 64 ? tile_group<64>(part, a, splits, stream) : tile_group<128>(part, a, splits, stream);
    }
    if (e != cudaSuccess) { set_cuda_error(e, "int4_tile launch"); return PGB_ERR_CUDA; }
    return check_launch("int4_tile_kernel");
}

int int4_tile_error_flag(int *out) { return tc_read_error_flag(out); }

}  // namespace pgb
