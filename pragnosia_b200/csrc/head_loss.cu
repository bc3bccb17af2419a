// Losses straight from the hidden states and the head's weight, s_nv = h_n . w_v, without the (N, V) logits in memory: softmax
// cross entropy against a given word per row, and distillation from a teacher's top logits. Both are one operator: a row has a target
// distribution p over few words (one word of probability 1, or the teacher's k), a temperature tau, and
//     L_n = log2 sum_v 2^(a s_nv)                        a = log2(e) / tau
//     l_n = tau^2 (sum_j p log p + L_n ln 2) - tau sum_j p_nj s_{n,i_nj}
//     ds_nv = c_n tau (2^(a s_nv - L_n) - sum_{j: i_nj = v} p_nj),   dh = ds W,   dW = ds^T h.
// Forward: one product whose epilogue keeps, per row and 256-column tile, the running maximum and sum and the targets' logits; a
// second kernel joins the tiles of a row. Backward: the same product again, whose epilogue turns the tile into ds, rounded to bf16, in a
// workspace that holds a piece of the (N, V) matrix; behind it one launch multiplies the piece with W and with h. Arithmetic: 2 N V d
// forward, 6 N V d backward (a third of it the logits again, the price of not keeping them).
//   Pieces: along the longer of N and V, so that the gradient that gathers over pieces (fp32, added to in place) is the smaller one.
//   ds holds no upstream scale where that is the same for every row (mean, sum): the scale is applied to the fp32 accumulators.
//   Rounded to bf16, ds is off by 2^-9 of itself, as the gradients themselves are when they are bf16.
//   fp32 operands: three bf16 terms each (24 bits), six of the nine products (what is left out is below 2^-23 of the sum's terms), small
//   ones first, all into one accumulator; ds as three terms as well.
// The product: pairs of SMs, 256 x 256 tiles, tcgen05.mma.cta_group::2, six 32 KiB stages a CTA fed by TMA, two accumulators in tensor
// memory so that a tile's epilogue runs under the next one's products; 16 epilogue warps, a row and a column quarter each.
#include <math.h>

#include "tc_pair.cuh"

namespace pgb {

constexpr int HL_B = 256, HL_BK = 64, HL_STAGES = 6, HL_EPI = 16, HL_NT = (2 + HL_EPI) * 32;
constexpr int HL_HALF = (HL_B / 2) * HL_BK * 2, HL_STAGE = 2 * HL_HALF;     // a CTA's share of one operand's block, of both
constexpr int HL_CW = HL_B / (HL_EPI / 4);                            // columns of a tile that an epilogue warp owns
constexpr int HL_OUT_BYTES = 32 * 64;                                 // staging of an epilogue warp: 32 rows of 64 bytes
constexpr int HL_SMEM = HL_STAGES * HL_STAGE + 1024 + HL_EPI * HL_OUT_BYTES + 1024;
constexpr int HL_GROUP = 16;                                          // row blocks that a sweep over the columns takes together
constexpr long long HL_PIECE_BYTES = 96LL << 20;                      // of ds in the workspace at once: what stays in the 126 MB L2
static_assert(HL_STAGE % 1024 == 0 && HL_SMEM <= 232448, "shared memory");
constexpr float LOG2E_F = 1.4426950408889634f;

struct HlMaps { CUtensorMap a[2], b[2]; };
// An epilogue warp's share of a tile: rows row0 .. +31 (a lane each), columns col0 .. +63; block: which of the tile's 32 it is. t, k0, k1, kt: the
// tile and what of its K blocks the accumulator holds.
struct HlTile { int lane, sub, part, block, n, row0, col0, g, t, k0, k1, kt; uint32_t ti; };
// One product C[M][N] = A B^T over kb blocks of 64 (npairs times: the products of the operands' bf16 terms).
// a_mn / b_mn: the operand lies with its M / N axis contiguous instead of K.
struct HlProduct {
    int tiles_m = 0, tiles_n = 0, kb = 0, npairs = 1, a_mn = 0, b_mn = 0;
    __host__ __device__ int tiles() const { return tiles_m * tiles_n; }
    __host__ __device__ int kt() const { return kb * npairs; }
    // row blocks fastest, HL_GROUP of them at a time: B is read once per group, whatever its size
    __device__ void at(int t, int &m, int &n) const {
        const unsigned group = (unsigned)HL_GROUP * tiles_n, g = (unsigned)t / group, in = (unsigned)t - g * group;
        const unsigned gm = min(HL_GROUP, tiles_m - (int)g * HL_GROUP);
        n = in / gm;
        m = g * HL_GROUP + in - n * gm;
    }
};
// What a pair of SMs does: whole tiles, dealt out in turn (CUT false), or an equal share of all K blocks of both products, so that the first
// and the last tile of a share may be a part of one (CUT true).
template <bool CUT>
struct HlShare {
    const HlProduct *pr;
    int g = 0, t = 0, k0 = 0, k1 = 0, kt = 0;                         // the part at hand: product, tile, K blocks
    long long left = 0;
    static __host__ __device__ long long units(const HlProduct *pr) { return (long long)pr[0].tiles() * pr[0].kt() + (long long)pr[1].tiles() * pr[1].kt(); }
    static __device__ long long bound(long long total, int pair, int pairs) { return total / pairs * pair + total % pairs * pair / pairs; }
    // the pair whose share holds K block u
    static __device__ int owner(long long total, long long u, int pairs) {
        int q = (int)((double)u * pairs / (double)total);
        while (q + 1 < pairs && bound(total, q + 1, pairs) <= u) ++q;
        while (q > 0 && bound(total, q, pairs) > u) --q;
        return q;
    }
    __device__ HlShare(const HlProduct *pr, int pair, int pairs) : pr(pr) {
        if constexpr (CUT) {
            const long long total = units(pr), n0 = (long long)pr[0].tiles() * pr[0].kt(), from = bound(total, pair, pairs);
            left = bound(total, pair + 1, pairs) - from;
            g = from >= n0;
            kt = pr[g].kt();
            const long long in = g ? from - n0 : from;
            t = kt > 0 ? (int)(in / kt) : 0;
            k0 = kt > 0 ? (int)(in - (long long)t * kt) : 0;
            k1 = (int)(kt - k0 < left ? kt : k0 + left);
        } else {
            t = pair; kt = k1 = pr[0].kt();
            left = t < pr[0].tiles();
        }
    }
    __device__ bool more() const { return left > 0; }
    __device__ void next(int pairs) {
        if constexpr (CUT) {
            left -= k1 - k0;
            if (++t == pr[g].tiles() && g == 0) { g = 1; t = 0; kt = pr[1].kt(); }
            k0 = 0;
            k1 = (int)(kt < left ? kt : left);
        } else {
            t += pairs;
            left = t < pr[0].tiles();
        }
    }
};
// the terms of the two operands that product number pp of npairs multiplies (0: the head), small products first
__device__ __forceinline__ void hl_terms(int pp, int npairs, int &ta, int &tb) {
    const int q = npairs == 1 ? 5 : pp;                               // (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
    ta = (0x001102 >> (4 * q)) & 15;
    tb = (0x010120 >> (4 * q)) & 15;
}

// The roles of the kernel. An epilogue warp takes its 32 x 64 block of a complete accumulator into registers, hands the accumulator back at once, and
// works on them while what the next tile needs of its rows (epi.fetch) is on its way.
template <bool CUT, class Epi>
__device__ __forceinline__ void hl_body(const HlMaps &maps, const HlProduct *pr, Epi &epi) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;      // the same offset in both CTAs: one descriptor serves both
    uint8_t *sm = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t mb = base + HL_STAGES * HL_STAGE;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + HL_STAGES * HL_STAGE + 512);
    auto bar_full = [&](int s) { return mb + 8 * s; };                 // used in the first CTA only
    auto bar_empty = [&](int s) { return mb + 64 + 8 * s; };
    auto bar_acc_full = [&](int a) { return mb + 128 + 8 * a; };
    auto bar_acc_empty = [&](int a) { return mb + 144 + 8 * a; };      // used in the first CTA only
    auto bar_quarters = [&](int sub, int a) { return mb + 192 + 32 * sub + 8 * a; };   // three of a row's column quarters are in shared memory

    const int tid = threadIdx.x, lane = tid & 31, warp = warp_uniform(tid >> 5);
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (tid == 0) {
        for (int s = 0; s < HL_STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(bar_acc_full(a), 1); mbar_init(bar_acc_empty(a), 2 * HL_EPI); }
        for (int q = 0; q < 16; ++q) mbar_init(bar_quarters(q >> 2, q & 3), 3);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                                // the partner's barriers and tensor memory exist from here on
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    pdl_wait();
    pdl_launch_dependents();

    HlShare<CUT> w(pr, pair, pairs);
    int m, n;
    if (warp == 0) {
        // ------------------------------------------------------------------------------------------ producer (both CTAs)
        const bool leader = elect_one();
        uint32_t it = 0;
        bool ok = true;
        for (; w.more() && ok; w.next(pairs)) {
            const HlProduct &p = pr[w.g];
            p.at(w.t, m, n);
            const int m0 = m * HL_B + (int)rank * (HL_B / 2), n0 = n * HL_B + (int)rank * (HL_B / 2);
            const CUtensorMap *ma = &maps.a[w.g], *mbm = &maps.b[w.g];
            int pp = w.k0 / p.kb, kc = w.k0 - pp * p.kb, ta, tb;
            hl_terms(pp, p.npairs, ta, tb);
            for (int k = w.k0; k < w.k1 && ok; ++k, ++it) {
                const int s = it % HL_STAGES;
                if (it >= HL_STAGES) ok = __all_sync(0xffffffffu, mbar_wait(bar_empty(s), ((it / HL_STAGES) + 1) & 1, 91));
                if (ok && leader) {
                    const int c = kc * HL_BK;
                    const uint32_t sa = base + s * HL_STAGE, sb = sa + HL_HALF, full0 = cluster_addr(bar_full(s), 0);
                    if (rank == 0) mbar_expect_tx(bar_full(s), 2 * HL_STAGE);      // both CTAs' bytes
                    if (p.a_mn) {                                      // 64 rows of K, 64 contiguous rows of M at a time
                        lp_tma_load(sa, ma, full0, m0, c, ta);
                        lp_tma_load(sa + HL_HALF / 2, ma, full0, m0 + 64, c, ta);
                    } else {
                        lp_tma_load(sa, ma, full0, c, m0, ta);
                    }
                    if (p.b_mn) {
                        lp_tma_load(sb, mbm, full0, n0, c, tb);
                        lp_tma_load(sb + HL_HALF / 2, mbm, full0, n0 + 64, c, tb);
                    } else {
                        lp_tma_load(sb, mbm, full0, c, n0, tb);
                    }
                }
                if (++kc == p.kb) { kc = 0; hl_terms(++pp, p.npairs, ta, tb); }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------------------------------ MMA issuer (first CTA)
        if (rank == 0) {
            uint32_t it = 0, ti = 0;
            bool ok = true;
            for (; w.more() && ok; w.next(pairs), ++ti) {
                const int amn = pr[w.g].a_mn, bmn = pr[w.g].b_mn;
                const uint32_t idesc = idesc_bf16(HL_B, HL_B, amn, bmn), a = ti & 1;
                const uint32_t stepa = amn ? 128 : 2, stepb = bmn ? 128 : 2;
                if (ti >= 2) ok = __all_sync(0xffffffffu, lp_wait_cluster(bar_acc_empty(a), ((ti >> 1) + 1) & 1, 92));
                tc_fence_after();
                for (int k = w.k0; k < w.k1 && ok; ++k, ++it) {
                    const int s = it % HL_STAGES;
                    ok = __all_sync(0xffffffffu, lp_wait_cluster(bar_full(s), (it / HL_STAGES) & 1, 93));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = base + s * HL_STAGE;
                    const uint64_t da = smem_desc(sa, amn ? HL_HALF / 2 : 16, 1024), db = smem_desc(sa + HL_HALF, bmn ? HL_HALF / 2 : 16, 1024);
#pragma unroll
                    for (int q = 0; q < HL_BK / 16; ++q) lp_mma_elect(tmem + a * HL_B, da + q * stepa, db + q * stepb, idesc, (k > w.k0) | (q > 0));
                    lp_commit_elect(bar_empty(s));                     // the stage is free in both CTAs once these MMAs have read it
                    lp_commit_elect(cluster_addr(bar_empty(s), 1));
                }
                if (ok) {
                    lp_commit_elect(bar_acc_full(a));
                    lp_commit_elect(cluster_addr(bar_acc_full(a), 1));
                }
            }
        }
    } else {
        // ------------------------------------------------------------------------------------------ epilogue (both CTAs)
        const int sub = warp & 3, part = (warp - 2) >> 2;
        const uint32_t lane_base = (uint32_t)(32 * sub) << 16, acc_empty0 = cluster_addr(bar_acc_empty(0), 0), acc_empty1 = cluster_addr(bar_acc_empty(1), 0);
        uint8_t *stage = sm + HL_STAGES * HL_STAGE + 1024 + (warp - 2) * HL_OUT_BYTES, *shared = sm + HL_STAGES * HL_STAGE + 1024;
        const int row_in = (int)rank * (HL_B / 2) + 32 * sub, col_in = part * HL_CW;
        HlTile x;
        x.lane = lane; x.sub = sub; x.part = part; x.block = (int)rank * HL_EPI + (warp - 2);
        uint32_t ti = 0;
        bool ok = w.more();
        if (ok) {
            pr[w.g].at(w.t, m, n);
            epi.fetch(m * HL_B + row_in + lane, n * HL_B + col_in);
        }
        for (; ok; ++ti) {
            const uint32_t a = ti & 1;
            x.n = n; x.row0 = m * HL_B + row_in; x.col0 = n * HL_B + col_in; x.ti = ti;
            x.g = w.g; x.t = w.t; x.k0 = w.k0; x.k1 = w.k1; x.kt = w.kt;
            epi.begin(x);
            ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_full(a), (ti >> 1) & 1, 94));
            if (!ok) break;
            tc_fence_after();
            float v[2][32];
            const uint32_t tacc = tmem + lane_base + a * HL_B + part * HL_CW;
            tmem_ld32_nowait(tacc, v[0]);
            tmem_ld32_nowait(tacc + 32, v[1]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 64; ++i) asm volatile("" : "+f"(v[i >> 5][i & 31]));      // nothing that uses them moves ahead of the wait
            tc_fence_before();
            __syncwarp();
            if (lane == 0) lp_arrive_cluster(a ? acc_empty1 : acc_empty0);
            w.next(pairs);
            const bool more = w.more();
            if (more) {
                pr[w.g].at(w.t, m, n);
                epi.fetch(m * HL_B + row_in + lane, n * HL_B + col_in);
            }
            ok = epi.tile(x, v, stage, shared, bar_quarters(sub, ti & 3)) && more;
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();                                                // neither CTA frees tensor memory the other's MMAs may still write
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// v[i] for an i of each lane's own: a tree of selects keeps v in registers
__device__ __forceinline__ float pick32(const float (&v)[32], int i) {
    float a[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) a[j] = (i & 16) ? v[j + 16] : v[j];
#pragma unroll
    for (int w = 8; w > 0; w >>= 1)
#pragma unroll
        for (int j = 0; j < w; ++j) a[j] = (i & w) ? a[j + w] : a[j];
    return a[0];
}

// What a row's target distribution is read from: a word per row (target), or a list of k (ids ascending, INT_MAX behind the last entry;
// p their probabilities; ent the sum of p log p, NaN where an id was out of range).
struct HlTargets {
    const long long *target; long long ignore; const int *ids; const float *p, *ent; int k;
};

// A lane's walk over its row's targets: nx is the column of the one to come (INT_MAX: none), in ascending order.
template <bool LIST>
struct HlWalk {
    int nx = 0x7fffffff, pos = 0, k = 0;
    const int *ids = nullptr; const float *p = nullptr;
    // the targets from column `from` (of the whole vocabulary) on; word: the row's target; row < 0: none
    __device__ __forceinline__ void begin(const HlTargets &t, long long row, long long word, int from) {
        nx = 0x7fffffff;
        if (row < 0) return;
        if constexpr (LIST) {
            k = t.k; ids = t.ids + row * k; p = t.p + row * k;
            int lo = 0, hi = k;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ids[mid] < from) lo = mid + 1; else hi = mid;
            }
            pos = lo;
            if (pos < k) nx = ids[pos];
        } else {
            if (word != t.ignore && word >= from && word < 0x7fffffff) nx = (int)word;
        }
    }
    __device__ __forceinline__ float weight() const { return LIST ? p[pos] : 1.0f; }
    __device__ __forceinline__ void advance() {
        if constexpr (LIST) { ++pos; nx = pos < k ? ids[pos] : 0x7fffffff; } else nx = 0x7fffffff;
    }
};

// ------------------------------------------------------------------------------------------------ forward
struct HlFwd {
    HlTargets t; float a;
    float2 *ml;                                                       // [tiles_n][Np]: maximum (times a) and sum of a tile's row
    float *dot;                                                       // list: [tiles_n][Np], sum of p s over the tile; else [N], the target's s
    unsigned *ticket; long long N, Np; int V;
};
template <bool LIST>
struct HlFwdEpi {
    const HlFwd &f;
    HlWalk<LIST> w;
    long long row, word;                                               // of the tile fetched for
    __device__ __forceinline__ void fetch(int r, int) {
        row = r < f.N ? r : -1;
        if (!LIST) word = row >= 0 ? f.t.target[row] : f.t.ignore;
    }
    __device__ __forceinline__ void begin(const HlTile &x) { w.begin(f.t, row, word, x.col0); }
    __device__ __forceinline__ bool tile(const HlTile &x, float (&v)[2][32], uint8_t *, uint8_t *shared, uint32_t quarters) {
        float m = -INFINITY, l = 0.f, dot = 0.f;
        const int row = x.row0 + x.lane;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int c0 = x.col0 + 32 * b;
            if (c0 >= f.V) break;
            while (__any_sync(0xffffffffu, w.nx < c0 + 32)) {          // this block holds a target of some row
                const bool hit = w.nx < c0 + 32;
                const float s = pick32(v[b], hit ? w.nx - c0 : 0);
                if (hit) { dot = fmaf(w.weight(), s, dot); w.advance(); if (!LIST) f.dot[row] = s; }
            }
            if (c0 + 32 > f.V) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[b][i] = c0 + i < f.V ? v[b][i] : -INFINITY;
            }
            float t4[4] = {v[b][0], v[b][1], v[b][2], v[b][3]};
#pragma unroll
            for (int i = 4; i < 32; ++i) t4[i & 3] = fmaxf(t4[i & 3], v[b][i]);
            const float top = fmaxf(m, f.a * fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
            const float at = top == -INFINITY ? 0.f : top;
            float s4[4] = {l * fast_exp2(m - at), 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 32; ++i) s4[i & 3] += fast_exp2(fmaf(v[b][i], f.a, -at));
            l = (s4[0] + s4[1]) + (s4[2] + s4[3]);
            m = top;
        }
        // The four column quarters of a row, by the first one's warp. Four sets in turn, each with a barrier: a warp has tile t + 3 in hand only
        // once every warp has taken tile t + 1 out of tensor memory, which is behind its work on tile t.
        float3 *mine = reinterpret_cast<float3 *>(shared) + ((x.ti & 3) * 128 + 32 * x.sub + x.lane) * 4;
        if (x.part != 0) {
            mine[x.part] = make_float3(m, l, dot);
            __syncwarp();
            if (x.lane == 0) mbar_arrive(quarters);
            return true;
        }
        const bool ok = mbar_wait_warp(quarters, (x.ti >> 2) & 1, 95);
        if (ok) {
#pragma unroll
            for (int q = 1; q < 4; ++q) {
                const float3 o = mine[q];
                const float top = fmaxf(m, o.x), at = top == -INFINITY ? 0.f : top;
                l = l * fast_exp2(m - at) + o.y * fast_exp2(o.x - at);
                m = top;
                dot += o.z;
            }
            if (row < f.N) {
                f.ml[(long long)x.n * f.Np + row] = make_float2(m, l);
                if (LIST) f.dot[(long long)x.n * f.Np + row] = dot;
            }
        }
        return ok;
    }
};
template <bool LIST>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HL_NT, 1)
head_loss_fwd_kernel(const __grid_constant__ HlMaps maps, const __grid_constant__ HlProduct pr, const __grid_constant__ HlFwd f) {
    if (blockIdx.x == 0 && threadIdx.x == 0) { pdl_wait(); *f.ticket = 0u; }
    HlFwdEpi<LIST> epi{f, {}, 0, 0};
    hl_body<false>(maps, &pr, epi);
}

// Joins a row's tiles: 32 rows a block (a lane each), the tiles dealt out to its 8 warps, then the block's losses and live rows as one
// partial sum; the last block to finish adds the partials up in order, so the sum does not depend on who that is.
struct HlJoin {
    HlTargets t; const float2 *ml; const float *dot; float2 *L; float *row_loss, *loss, *count; double2 *partial; unsigned *ticket;
    long long N, Np; int V, tiles; float tau; int reduction;
};
template <bool LIST>
__global__ void __launch_bounds__(256) head_loss_join_kernel(const HlJoin j) {
    __shared__ float3 part[8][32];
    __shared__ double2 sums[8];
    __shared__ bool last;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * 32 + lane;
    float m = -INFINITY, l = 0.f, dot = 0.f;
    if (row < j.N) {
#pragma unroll 4
        for (int n = warp; n < j.tiles; n += 8) {
            const float2 o = j.ml[(long long)n * j.Np + row];
            const float top = fmaxf(m, o.x), at = top == -INFINITY ? 0.f : top;
            l = l * fast_exp2(m - at) + o.y * fast_exp2(o.x - at);
            m = top;
            if (LIST) dot += j.dot[(long long)n * j.Np + row];
        }
    }
    part[warp][lane] = make_float3(m, l, dot);
    __syncthreads();
    double loss = 0.0;
    bool live = false;
    if (warp == 0 && row < j.N) {
        double sum = l, d = dot;
        for (int q = 1; q < 8; ++q) {
            const float3 o = part[q][lane];
            const float top = fmaxf(m, o.x), at = top == -INFINITY ? 0.f : top;
            sum = sum * exp2((double)m - at) + o.y * exp2((double)o.x - at);
            m = top;
            d += o.z;
        }
        const double L = (double)m + log2(sum);
        const float hi = (float)L;
        j.L[row] = make_float2(hi, (float)(L - hi));
        if (LIST) {
            const float ent = j.t.ent[row];
            live = j.t.ids[row * j.t.k] != 0x7fffffff || ent != ent;
            loss = (double)j.tau * j.tau * (ent + L * 0.693147180559945309) - j.tau * d;
        } else {
            const long long w = j.t.target[row];
            live = w != j.t.ignore;
            loss = live && w >= 0 && w < j.V ? L * 0.693147180559945309 - j.dot[row] : NAN;
        }
        if (!live) loss = 0.0;
        if (j.row_loss) j.row_loss[row] = (float)loss;
    }
    if (j.reduction == 0) return;
    if (warp == 0) {
        double c = live;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            loss += __shfl_xor_sync(0xffffffffu, loss, o);
            c += __shfl_xor_sync(0xffffffffu, c, o);
        }
        if (lane == 0) {
            j.partial[blockIdx.x] = make_double2(loss, c);
            __threadfence();
            last = atomicAdd(j.ticket, 1u) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double2 s = make_double2(0.0, 0.0);
    for (unsigned b = threadIdx.x; b < gridDim.x; b += 256) {
        const double2 o = __ldcg(j.partial + b);
        s.x += o.x; s.y += o.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { s.x += __shfl_xor_sync(0xffffffffu, s.x, o); s.y += __shfl_xor_sync(0xffffffffu, s.y, o); }
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int q = 1; q < 8; ++q) { s.x += sums[q].x; s.y += sums[q].y; }
        *j.loss = (float)(j.reduction == 2 ? s.x / s.y : s.x);
        *j.count = (float)s.y;
    }
}

// ------------------------------------------------------------------------------------------------ a teacher's lists
// A warp per row: probabilities of the entries that are there (id >= 0, logit not -inf) at the temperature, in ascending order of their
// ids (a rank per entry: k comparisons each).
__global__ void __launch_bounds__(128) head_teacher_kernel(const long long *__restrict__ in_ids, const float *__restrict__ in_logits, int *__restrict__ ids,
                                                           float *__restrict__ p, float *__restrict__ ent, long long N, int V, int k, float inv_tau) {
    extern __shared__ int teacher_smem[];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= N) return;
    int *id = teacher_smem + 2 * k * warp;
    float *z = reinterpret_cast<float *>(id + k);
    float top = -INFINITY;
    bool bad = false;
    for (int j = lane; j < k; j += 32) {
        const long long i = in_ids[row * k + j];
        const float x = in_logits[row * k + j] * inv_tau;
        const bool here = i >= 0 && x != -INFINITY;
        bad |= here && i >= V;
        id[j] = here ? (i >= V ? V : (int)i) : 0x7fffffff;
        z[j] = here ? x : -INFINITY;
        if (here) top = fmaxf(top, x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad = __any_sync(0xffffffffu, bad);
    __syncwarp();
    float sum = 0.f;
    for (int j = lane; j < k; j += 32)
        if (id[j] != 0x7fffffff) sum += expf(z[j] - top);
    sum = warp_sum(sum);
    float e = 0.f;
    for (int j = lane; j < k; j += 32) {
        const int me = id[j];
        const bool here = me != 0x7fffffff;
        const float q = here ? expf(z[j] - top) / sum : 0.f;
        if (here && !(q <= 0.f)) e += q * ((z[j] - top) - logf(sum));  // NaN stays
        int rank = 0;
        for (int i = 0; i < k; ++i) rank += id[i] < me || (id[i] == me && i < j);
        ids[row * k + rank] = me;
        p[row * k + rank] = q;
    }
    e = warp_sum(e);
    if (lane == 0) ent[row] = bad ? NAN : e;
}

// ------------------------------------------------------------------------------------------------ backward
struct HlProb {
    HlTargets t; const float2 *L; const float *row_weight;            // row_weight NULL: 1
    float a; __nv_bfloat16 *P; long long ldp, part_stride;            // P [terms][rows of the piece][ldp]
    long long row_from; int V, col_from, cols, rows;                  // the piece: rows and columns it begins at, how many
    unsigned *tickets; int n_tickets;                                 // set to zero for the products behind
};
template <bool LIST, int TERMS>
struct HlProbEpi {
    const HlProb &f;
    HlWalk<LIST> w;
    long long row, word; float2 L; float weight, ent; int id0;         // of the tile fetched for
    float a_hi, a_lo, c; bool live;                                   // of the tile at hand
    __device__ __forceinline__ void fetch(int r, int) {
        row = r < f.rows ? f.row_from + r : -1;
        if (row < 0) return;
        L = f.L[row];
        weight = f.row_weight ? f.row_weight[row] : 1.f;
        if (LIST) { ent = f.t.ent[row]; id0 = f.t.ids[row * f.t.k]; } else word = f.t.target[row];
    }
    __device__ __forceinline__ void begin(const HlTile &x) {
        w.begin(f.t, row, word, f.col_from + x.col0);
        a_hi = -L.x; a_lo = -L.y;
        const bool bad = LIST ? ent != ent : word != f.t.ignore && (word < 0 || word >= f.V);
        live = row >= 0 && (LIST ? bad || id0 != 0x7fffffff : word != f.t.ignore);
        c = bad ? NAN : weight;
    }
    __device__ __forceinline__ bool tile(const HlTile &x, float (&vv)[2][32], uint8_t *stage, uint8_t *, uint32_t) {
        const int lane = x.lane;
        // 64-byte rows, their 16-byte chunks rotated by the row: the row-per-lane writes and the chunk-per-lane reads both touch every bank once
        auto chunk_at = [&](int r, int ch) { return stage + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4); };
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int c0 = x.col0 + 32 * b, v0 = f.col_from + c0;
            if (c0 >= f.cols) break;
            float (&v)[32] = vv[b];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = TERMS == 3 ? fast_exp2(fmaf(v[i], f.a, a_hi) + a_lo) : fast_exp2(fmaf(v[i], f.a, a_hi));
            while (__any_sync(0xffffffffu, w.nx < v0 + 32)) {
                const bool hit = w.nx < v0 + 32;
                const int at = hit ? w.nx - v0 : -1;
                const float less = hit ? w.weight() : 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= i == at ? less : 0.f;
                if (hit) w.advance();
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = live ? c * v[i] : 0.f;
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    __nv_bfloat162 o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        o[i] = __floats2bfloat162_rn(v[8 * ch + 2 * i], v[8 * ch + 2 * i + 1]);
                        if (term + 1 < TERMS) {
                            const float2 h = __bfloat1622float2(o[i]);
                            v[8 * ch + 2 * i] -= h.x; v[8 * ch + 2 * i + 1] -= h.y;
                        }
                    }
                    *reinterpret_cast<uint4 *>(chunk_at(lane, ch)) = *reinterpret_cast<uint4 *>(o);
                }
                __syncwarp();
                __nv_bfloat16 *P = f.P + term * f.part_stride;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int r = (lane >> 2) + 8 * q, ch = lane & 3;
                    const uint4 val = *reinterpret_cast<const uint4 *>(chunk_at(r, ch));
                    if (x.row0 + r < f.rows && c0 + 8 * ch < f.ldp) *reinterpret_cast<uint4 *>(P + (long long)(x.row0 + r) * f.ldp + c0 + 8 * ch) = val;
                }
                __syncwarp();
            }
        }
        return true;
    }
};
template <bool LIST, int TERMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HL_NT, 1)
head_loss_ds_kernel(const __grid_constant__ HlMaps maps, const __grid_constant__ HlProduct pr, const __grid_constant__ HlProb f) {
    pdl_wait();
    for (int i = blockIdx.x * HL_NT + threadIdx.x; i < f.n_tickets; i += gridDim.x * HL_NT) f.tickets[i] = 0u;
    HlProbEpi<LIST, TERMS> epi{f};
    hl_body<false>(maps, &pr, epi);
}

// The upstream scale that all rows share: g the gradient of the (summed or averaged) loss, count the rows averaged over.
__device__ __forceinline__ float hl_alpha(const float *g, const float *count, float tau, int reduction) {
    if (reduction == 0) return tau;
    if (reduction == 1) return tau * *g;
    const float n = *count;
    return n > 0.f ? tau * *g / n : 0.f;                              // no row counts: no gradient (the loss itself is 0 / 0)
}
// What becomes of a product's tiles: out = alpha * (acc +) C, or acc (+)= C where further pieces follow. acc [rows][d] fp32.
struct HlGrad { float *acc; void *out; long long rows; int adds, last; };
struct HlGrads {
    HlGrad g[2]; const float *up, *count; float tau; int reduction, d, out_f32;
    float *parts; unsigned *tickets;                                  // parts [pairs][2][32][2048]: what pairs hold of cut tiles
};
// A tile that shares cut is summed by whoever finishes it last (each of its 32 blocks by itself): the others have left their parts in
// memory, and all are added in the order of K, so the sum does not depend on who that is.
struct HlGradEpi {
    const HlGrads &f;
    const HlProduct *pr;
    float alpha;
    __device__ __forceinline__ void fetch(int, int) {}
    __device__ __forceinline__ void begin(const HlTile &) {}
    __device__ __forceinline__ float4 *part_of(int pair, bool head, int block, int lane) const {
        return reinterpret_cast<float4 *>(f.parts) + (((long long)pair * 2 + head) * 32 + block) * 512 + lane;
    }
    __device__ __forceinline__ bool tile(const HlTile &x, float (&v)[2][32], uint8_t *stage, uint8_t *, uint32_t) {
        const HlGrad &o = f.g[x.g];
        const int lane = x.lane;
        if (x.col0 >= f.d || x.row0 >= o.rows) return true;           // nothing of the matrix in this block; its ticket is not drawn by anyone
        if (x.k1 - x.k0 < x.kt) {
            const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
            float4 *mine = part_of(pair, x.k0 == 0, x.block, lane);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float *s = &v[j >> 3][4 * (j & 7)];
                mine[32 * j] = make_float4(s[0], s[1], s[2], s[3]);
            }
            const long long total = HlShare<true>::units(pr), from = (x.g ? (long long)pr[0].tiles() * pr[0].kt() : 0) + (long long)x.t * x.kt;
            const int q0 = HlShare<true>::owner(total, from, pairs), q1 = HlShare<true>::owner(total, from + x.kt - 1, pairs);
            __threadfence();
            __syncwarp();
            unsigned before = 0;
            if (lane == 0) before = atomicAdd(f.tickets + ((long long)(x.g ? pr[0].tiles() : 0) + x.t) * 32 + x.block, 1u);
            before = __shfl_sync(0xffffffffu, before, 0);
            if (before != (unsigned)(q1 - q0)) return true;
            __threadfence();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float4 a = __ldcg(part_of(q0, true, x.block, lane) + 32 * j);
                float *s = &v[j >> 3][4 * (j & 7)];
                s[0] = a.x; s[1] = a.y; s[2] = a.z; s[3] = a.w;
            }
            for (int q = q0 + 1; q <= q1; ++q) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    const float4 a = __ldcg(part_of(q, false, x.block, lane) + 32 * j);
                    float *s = &v[j >> 3][4 * (j & 7)];
                    s[0] += a.x; s[1] += a.y; s[2] += a.z; s[3] += a.w;
                }
            }
        }
        auto chunk_at = [&](int r, int ch) { return stage + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4); };
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int c0 = x.col0 + 16 * b;
            if (c0 >= f.d) break;
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
                const float *s = &v[b >> 1][16 * (b & 1) + 4 * ch];
                *reinterpret_cast<float4 *>(chunk_at(lane, ch)) = make_float4(s[0], s[1], s[2], s[3]);
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = (lane >> 2) + 8 * q, ch = lane & 3, col = c0 + 4 * ch;
                float4 val = *reinterpret_cast<const float4 *>(chunk_at(r, ch));
                if (x.row0 + r < o.rows && col < f.d) {
                    const long long at = (long long)(x.row0 + r) * f.d + col;
                    if (o.adds) {
                        const float4 old = *reinterpret_cast<const float4 *>(o.acc + at);
                        val.x += old.x; val.y += old.y; val.z += old.z; val.w += old.w;
                    }
                    if (!o.last) {
                        *reinterpret_cast<float4 *>(o.acc + at) = val;
                    } else {
                        val.x *= alpha; val.y *= alpha; val.z *= alpha; val.w *= alpha;
                        if (f.out_f32) {
                            *reinterpret_cast<float4 *>(static_cast<float *>(o.out) + at) = val;
                        } else {
                            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(val.x, val.y), __floats2bfloat162_rn(val.z, val.w)};
                            *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(o.out) + at) = *reinterpret_cast<uint2 *>(h);
                        }
                    }
                }
            }
            __syncwarp();
        }
        return true;
    }
};
struct HlPair { HlProduct p[2]; };
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HL_NT, 1)
head_loss_grad_kernel(const __grid_constant__ HlMaps maps, const __grid_constant__ HlPair pr, const __grid_constant__ HlGrads f) {
    HlGradEpi epi{f, pr.p, 0.f};
    if (threadIdx.x >= 64) { pdl_wait(); epi.alpha = hl_alpha(f.up, f.count, f.tau, f.reduction); }
    hl_body<true>(maps, pr.p, epi);
}
// x as three bf16 terms, [3][n]; eight values a thread (n a multiple of 8)
__global__ void __launch_bounds__(256) head_split_kernel(const float *__restrict__ x, __nv_bfloat16 *__restrict__ out, long long n) {
    pdl_wait();
    pdl_launch_dependents();
    for (long long i = 8 * ((long long)blockIdx.x * 256 + threadIdx.x); i < n; i += 2048LL * gridDim.x) {
        float v[8];
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x + i);
        *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(x + i + 4);
        uint4 hi, lo, rest;
        split8(v, hi, lo, rest);
        *reinterpret_cast<uint4 *>(out + i) = hi;
        *reinterpret_cast<uint4 *>(out + n + i) = lo;
        *reinterpret_cast<uint4 *>(out + 2 * n + i) = rest;
    }
}

// ------------------------------------------------------------------------------------------------ host
static inline long long hl_up(long long x, long long to) { return (x + to - 1) / to * to; }
static inline int hl_tiles(long long n) { return (int)((n + HL_B - 1) / HL_B); }

// resident pairs of a kernel on the current device (cached per device); 0 if the query fails
template <class K>
static int hl_pairs(K kernel, int which) {
    static int cached[64][8];
    int dev = 0, sms = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    if (dev < 64 && cached[dev][which] > 0) return cached[dev][which];
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, HL_SMEM) != cudaSuccess) return 0;
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(sms > 1 ? sms & ~1 : 2)); cfg.blockDim = dim3(HL_NT); cfg.dynamicSmemBytes = HL_SMEM;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 2; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
    if (dev < 64) cached[dev][which] = n;
    return n;
}
template <class K, class Pr, class Ar>
static int hl_launch(K kernel, int which, const char *name, const HlMaps &maps, const Pr &pr, long long most, const Ar &args, cudaStream_t stream) {
    const int room = hl_pairs(kernel, which);
    if (room < 1) { set_cuda_error(cudaGetLastError(), name); return PGB_ERR_CUDA; }
    const unsigned pairs = (unsigned)(most < room ? most : room);
    cudaError_t e = pdl_launch(kernel, dim3(2 * pairs), dim3(HL_NT), (size_t)HL_SMEM, stream, maps, pr, args);
    if (e != cudaSuccess) { set_cuda_error(e, name); return PGB_ERR_CUDA; }
    return check_launch(name);
}

// an operand of the products: its first element, terms (1: the caller's bf16; 3: split), the elements between terms, rows' pitch
struct HlOperand { const void *ptr; int terms; long long term_stride, ld; };
// rows x cols of it as K-major blocks of 128 x 64, or as 64 x 64 ones whose columns are M or N
static bool hl_map(CUtensorMap *m, const HlOperand &o, long long row_from, long long col_from, long long rows, long long cols, bool mn) {
    const char *p = static_cast<const char *>(o.ptr) + 2 * (row_from * o.ld + col_from);
    return tc_make_map(m, p, o.terms, rows, cols, o.ld, o.terms > 1 ? o.term_stride : rows * o.ld, mn ? 64 : 128);
}

struct HlFwdPlan { long long Np, tiles, off_ml, off_dot, off_partial, off_ticket, off_h, off_w, total; };
static HlFwdPlan hl_fwd_plan(long long N, int V, int d, int dtype, bool list) {
    HlFwdPlan p;
    p.Np = hl_up(N, 32); p.tiles = hl_tiles(V);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += hl_up(bytes, 256); return o; };
    p.off_ml = take(p.tiles * p.Np * 8);
    p.off_dot = take((list ? p.tiles : 1) * p.Np * 4);
    p.off_partial = take(p.Np / 32 * 16);
    p.off_ticket = take(4);
    p.off_h = dtype == PGB_F32 ? take(6 * N * d) : 0;
    p.off_w = dtype == PGB_F32 ? take(6LL * V * d) : 0;
    p.total = at;
    return p;
}
long long head_loss_fwd_bytes(long long N, int V, int d, int dtype, int k) { return hl_fwd_plan(N, V, d, dtype, k > 0).total; }

static int hl_split(const void *x, void *out, long long n, cudaStream_t stream) {
    const long long blocks = (n / 8 + 255) / 256;
    cudaError_t e = pdl_launch(head_split_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, static_cast<const float *>(x),
                               static_cast<__nv_bfloat16 *>(out), n);
    if (e != cudaSuccess) { set_cuda_error(e, "head_split launch"); return PGB_ERR_CUDA; }
    return check_launch("head_split_kernel");
}
// the operand as the products take it; fp32: split into `room` first
static int hl_operand(HlOperand &o, const void *x, int dtype, long long rows, int d, void *room, cudaStream_t stream) {
    o = {x, 1, 0, d};
    if (dtype != PGB_F32) return PGB_OK;
    o = {room, 3, rows * d, d};
    return hl_split(x, room, rows * d, stream);
}
static int hl_no_map() { set_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled"); return PGB_ERR_CUDA; }

int head_teacher_launch(const long long *in_ids, const float *in_logits, int *ids, float *p, float *ent, long long N, int V, int k, float tau,
                        cudaStream_t stream) {
    cudaError_t e = pdl_launch(head_teacher_kernel, dim3((unsigned)((N + 3) / 4)), dim3(128), (size_t)(4 * k * 8), stream, in_ids, in_logits, ids, p, ent, N, V,
                               k, 1.0f / tau);
    if (e != cudaSuccess) { set_cuda_error(e, "head_teacher launch"); return PGB_ERR_CUDA; }
    return check_launch("head_teacher_kernel");
}

int head_loss_fwd_launch(const HeadLossArgs &x, float *row_loss, float *loss, float *count, float *L, void *scratch, cudaStream_t stream) {
    const bool list = x.ids != nullptr;
    const HlFwdPlan pl = hl_fwd_plan(x.N, x.V, x.d, x.dtype, list);
    char *s = static_cast<char *>(scratch);
    HlOperand h, w;
    int rc = hl_operand(h, x.h, x.dtype, x.N, x.d, s + pl.off_h, stream);
    if (rc == PGB_OK) rc = hl_operand(w, x.W, x.dtype, x.V, x.d, s + pl.off_w, stream);
    if (rc != PGB_OK) return rc;
    HlMaps maps;
    if (!hl_map(&maps.a[0], h, 0, 0, x.N, x.d, false) || !hl_map(&maps.b[0], w, 0, 0, x.V, x.d, false)) return hl_no_map();
    maps.a[1] = maps.a[0]; maps.b[1] = maps.b[0];
    HlProduct pr;
    pr.tiles_m = hl_tiles(x.N); pr.tiles_n = (int)pl.tiles; pr.kb = (x.d + HL_BK - 1) / HL_BK; pr.npairs = h.terms == 3 ? 6 : 1;
    const HlTargets t{x.target, x.ignore, x.ids, x.p, x.ent, x.k};
    const HlFwd f{t, LOG2E_F / x.tau, reinterpret_cast<float2 *>(s + pl.off_ml), reinterpret_cast<float *>(s + pl.off_dot),
                  reinterpret_cast<unsigned *>(s + pl.off_ticket), x.N, pl.Np, x.V};
    rc = list ? hl_launch(head_loss_fwd_kernel<true>, 0, "head_loss_fwd_kernel", maps, pr, pr.tiles(), f, stream)
              : hl_launch(head_loss_fwd_kernel<false>, 1, "head_loss_fwd_kernel", maps, pr, pr.tiles(), f, stream);
    if (rc != PGB_OK) return rc;
    const HlJoin j{t, f.ml, f.dot, reinterpret_cast<float2 *>(L), row_loss, loss, count, reinterpret_cast<double2 *>(s + pl.off_partial), f.ticket,
                   x.N, pl.Np, x.V, (int)pl.tiles, x.tau, x.reduction};
    cudaError_t e = pdl_launch(list ? head_loss_join_kernel<true> : head_loss_join_kernel<false>, dim3((unsigned)(pl.Np / 32)), dim3(256), 0, stream, j);
    if (e != cudaSuccess) { set_cuda_error(e, "head_loss_join launch"); return PGB_ERR_CUDA; }
    return check_launch("head_loss_join_kernel");
}

// How the backward pass is cut: pieces of `step` rows (by_rows) or columns.
struct HlBwdPlan {
    bool by_rows; long long step, pieces, ldp, rows, cols; int terms, pairs;   // pairs: that the products are shared out to at most
    long long off_p, off_acc, off_parts, off_tickets, off_h, off_w, total;
};
constexpr int HL_LEAST = 8;                                           // K blocks a pair takes at least: with fewer its parts cost more than its products
static HlBwdPlan hl_bwd_plan(long long N, int V, int d, int dtype, bool dh, bool dw) {
    HlBwdPlan p;
    p.terms = dtype == PGB_F32 ? 3 : 1;
    p.by_rows = N >= V;
    const long long most = HL_PIECE_BYTES / (2 * p.terms), across = hl_up(p.by_rows ? V : N, 64), along = p.by_rows ? N : V;
    long long step = most / across / HL_B * HL_B;
    if (step < HL_B) step = HL_B;
    p.pieces = (along + step - 1) / step;
    p.step = hl_up((along + p.pieces - 1) / p.pieces, HL_B);
    p.pieces = (along + p.step - 1) / p.step;
    p.ldp = p.by_rows ? hl_up(V, 64) : p.step;
    p.rows = p.by_rows && p.step < N ? p.step : N;
    p.cols = !p.by_rows && p.step < V ? p.step : V;
    const long long units = (long long)hl_tiles(d) * (p.terms == 3 ? 6 : 1) * (hl_tiles(p.rows) * hl_up(p.cols, HL_BK) + hl_tiles(p.cols) * hl_up(p.rows, HL_BK)) / HL_BK;
    p.pairs = sm_count() / 2;
    if (units / HL_LEAST < p.pairs) p.pairs = units / HL_LEAST < 1 ? 1 : (int)(units / HL_LEAST);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += hl_up(bytes, 256); return o; };
    p.off_p = take(2 * p.terms * p.rows * p.ldp);
    p.off_acc = p.pieces > 1 && (p.by_rows ? dw : dh) ? take(4 * (p.by_rows ? (long long)V : N) * d) : -1;   // of the gradient that gathers over pieces
    p.off_parts = take((long long)p.pairs * 2 * 32 * 2048 * 4);
    p.off_tickets = take(4LL * 32 * ((long long)hl_tiles(p.rows) + hl_tiles(p.cols)) * hl_tiles(d));
    p.off_h = dtype == PGB_F32 ? take(6 * N * d) : 0;
    p.off_w = dtype == PGB_F32 ? take(6LL * V * d) : 0;
    p.total = at;
    return p;
}
long long head_loss_bwd_bytes(long long N, int V, int d, int dtype, int want_dh, int want_dw) {
    return hl_bwd_plan(N, V, d, dtype, want_dh != 0, want_dw != 0).total;
}
int head_loss_bwd_launch(const HeadLossArgs &x, const float *L, const float *count, const float *up, void *dh, void *dw, void *scratch, cudaStream_t stream) {
    const bool list = x.ids != nullptr;
    const HlBwdPlan pl = hl_bwd_plan(x.N, x.V, x.d, x.dtype, dh != nullptr, dw != nullptr);
    char *s = static_cast<char *>(scratch);
    HlOperand h, w;
    int rc = hl_operand(h, x.h, x.dtype, x.N, x.d, s + pl.off_h, stream);
    if (rc == PGB_OK) rc = hl_operand(w, x.W, x.dtype, x.V, x.d, s + pl.off_w, stream);
    if (rc != PGB_OK) return rc;
    const int np = pl.terms == 3 ? 6 : 1, esize = x.dtype == PGB_F32 ? 4 : 2;
    const HlOperand P{s + pl.off_p, pl.terms, pl.rows * pl.ldp, pl.ldp};
    unsigned *tickets = reinterpret_cast<unsigned *>(s + pl.off_tickets);
    HlProb f{{x.target, x.ignore, x.ids, x.p, x.ent, x.k}, reinterpret_cast<const float2 *>(L), x.reduction == 0 ? up : nullptr, LOG2E_F / x.tau,
             reinterpret_cast<__nv_bfloat16 *>(s + pl.off_p), pl.ldp, pl.rows * pl.ldp, 0, x.V, 0, 0, 0, tickets, 0};
    HlGrads o{{}, up, count, x.tau, x.reduction, x.d, x.dtype == PGB_F32, reinterpret_cast<float *>(s + pl.off_parts), tickets};
    float *acc = pl.off_acc >= 0 ? reinterpret_cast<float *>(s + pl.off_acc) : nullptr;
    for (long long i = 0; i < pl.pieces; ++i) {
        const long long from = i * pl.step, row_from = pl.by_rows ? from : 0, col_from = pl.by_rows ? 0 : from;
        const long long rows = pl.by_rows ? (from + pl.step < x.N ? pl.step : x.N - from) : x.N;
        const long long cols = pl.by_rows ? x.V : (from + pl.step < x.V ? pl.step : x.V - from);
        const bool first = i == 0, last = i + 1 == pl.pieces;
        HlMaps maps;
        if (!hl_map(&maps.a[0], h, row_from, 0, rows, x.d, false) || !hl_map(&maps.b[0], w, col_from, 0, cols, x.d, false)) return hl_no_map();
        maps.a[1] = maps.a[0]; maps.b[1] = maps.b[0];
        HlPair two;
        if (dh) {                                                     // dh[rows] += P W[cols]
            HlProduct &q = two.p[0];
            q.tiles_m = hl_tiles(rows); q.tiles_n = hl_tiles(x.d); q.kb = (int)((cols + HL_BK - 1) / HL_BK); q.npairs = np; q.b_mn = 1;
            const bool gathers = !pl.by_rows && pl.pieces > 1;
            o.g[0] = {acc, static_cast<char *>(dh) + row_from * x.d * esize, rows, gathers && !first, !gathers || last};
        }
        if (dw) {                                                     // dW[cols] += P^T h[rows]
            HlProduct &q = two.p[1];
            q.tiles_m = hl_tiles(cols); q.tiles_n = hl_tiles(x.d); q.kb = (int)((rows + HL_BK - 1) / HL_BK); q.npairs = np; q.a_mn = 1; q.b_mn = 1;
            const bool gathers = pl.by_rows && pl.pieces > 1;
            o.g[1] = {acc, static_cast<char *>(dw) + col_from * x.d * esize, cols, gathers && !first, !gathers || last};
        }
        HlProduct pr;
        pr.tiles_m = hl_tiles(rows); pr.tiles_n = hl_tiles(cols); pr.kb = (x.d + HL_BK - 1) / HL_BK; pr.npairs = np;
        f.row_from = row_from; f.rows = (int)rows; f.col_from = (int)col_from; f.cols = (int)cols; f.n_tickets = 32 * (two.p[0].tiles() + two.p[1].tiles());
        if (pl.terms == 3)
            rc = list ? hl_launch(head_loss_ds_kernel<true, 3>, 2, "head_loss_ds_kernel", maps, pr, pr.tiles(), f, stream)
                      : hl_launch(head_loss_ds_kernel<false, 3>, 3, "head_loss_ds_kernel", maps, pr, pr.tiles(), f, stream);
        else
            rc = list ? hl_launch(head_loss_ds_kernel<true, 1>, 4, "head_loss_ds_kernel", maps, pr, pr.tiles(), f, stream)
                      : hl_launch(head_loss_ds_kernel<false, 1>, 5, "head_loss_ds_kernel", maps, pr, pr.tiles(), f, stream);
        if (rc != PGB_OK) return rc;
        if (dh && (!hl_map(&maps.a[0], P, 0, 0, rows, cols, false) || !hl_map(&maps.b[0], w, col_from, 0, cols, x.d, true))) return hl_no_map();
        if (dw && (!hl_map(&maps.a[1], P, 0, 0, rows, cols, true) || !hl_map(&maps.b[1], h, row_from, 0, rows, x.d, true))) return hl_no_map();
        long long pairs = HlShare<true>::units(two.p) / HL_LEAST;
        pairs = pairs < 1 ? 1 : pairs < pl.pairs ? pairs : pl.pairs;
        rc = hl_launch(head_loss_grad_kernel, 6, "head_loss_grad_kernel", maps, two, pairs, o, stream);
        if (rc != PGB_OK) return rc;
    }
    return PGB_OK;
}

int head_loss_error_flag(int *out) { return tc_read_error_flag(out); }

}  // namespace pgb
