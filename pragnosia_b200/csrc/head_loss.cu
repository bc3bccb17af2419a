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
//   A row that does not count has zeros in ds, but its h may hold what is no number, and zero times that is none either. The forward pass tells
// (such a row's sum of exponentials is no number), and the backward pass then multiplies a copy of h with zeros in those rows.
//   ds holds no upstream scale where that is the same for every row (mean, sum): the scale is applied to the fp32 accumulators.
//   Rounded to bf16, ds is off by at most 2^-8 of itself, as the gradients themselves are when they are bf16. Cross entropy's stay as near to 64 bits
// as fp32 logits take them (0.0017 in the 2-norm, their own rounding); distillation's, with several large entries a row, are at 0.0023.
//   What lies in memory beside operands and results. Forward: a tile row's maximum and sum, N V / 32 bytes, and of a teacher's lists the marks, N V / 4 (an
// eighth of bf16 logits). Backward: two pieces of ds, a clean copy of h, fp32 sums.
//   fp32 operands: three bf16 terms each (24 bits), six of the nine products (what is left out is below 2^-23 of the sum's terms); ds as
//   three terms as well. The tensor cores cut off what a partial sum has beyond fp32 instead of rounding it, so sums over a long K axis
//   drift (gradients were off by 5e-6 to 8e-6): there a block of 64 has an accumulator of its own, small products first, and the
//   blocks are added in registers.
// The product: pairs of SMs, 256 x 256 tiles, tcgen05.mma.cta_group::2, six 32 KiB stages a CTA fed by TMA, two accumulators in tensor
// memory so that a tile's epilogue runs under the next one's products; 16 epilogue warps, a row and a column quarter each.
//   What bounds it: the tensor pipe (97 % of a forward launch's active cycles and 91 % of its elapsed ones, 82 and 73 % of a backward one's), at the clock that the power limit leaves. 32768 rows, 8192
// words, 768 wide, bf16: forward 292 us (1.41 PFLOP/s), backward 1.09 ms (1.13 PFLOP/s; a launch's two ends are a tenth of it); fp32, 2000 rows, 704 wide: both 502 us.
#include <math.h>

#include "tc_pair.cuh"

namespace pgb {

constexpr int HL_B = 256, HL_BK = 64, HL_STAGES = 6, HL_EPI = 16, HL_NT = (2 + HL_EPI) * 32;
constexpr int HL_HALF = (HL_B / 2) * HL_BK * 2, HL_STAGE = 2 * HL_HALF;     // a CTA's share of one operand's block, of both
constexpr int HL_CW = HL_B / (HL_EPI / 4);                            // columns of a tile that an epilogue warp owns
constexpr int HL_OUT_BYTES = 32 * 64;                                 // staging of an epilogue warp: 32 rows of 64 bytes
constexpr int HL_SMEM = HL_STAGES * HL_STAGE + 1024 + HL_EPI * HL_OUT_BYTES + 1024;
constexpr int HL_GROUP = 16;                                          // row blocks that a sweep over the columns takes together
constexpr long long HL_PIECE_BYTES = 64LL << 20;                      // of ds, two such pieces in the workspace: one written, one read
static_assert(HL_STAGE % 1024 == 0 && HL_SMEM <= 232448, "shared memory");
constexpr float LOG2E_F = 1.4426950408889634f;

struct HlMaps { CUtensorMap a[3], b[3], ds, clean; };                 // of the products; ds: the piece of it that is written; clean: b[1] where *dirty is set
// An epilogue warp's share of a tile: rows row0 .. +31 (a lane each), columns col0 .. +63. g, sp: the product and the part of K that the accumulator
// holds; ti: how many tiles came before.
struct HlTile { int lane, sub, part, n, row0, col0, g, sp; uint32_t ti; };
// One product C[M][N] = A B^T over kb blocks of 64, its K axis in `splits` parts.
// a_mn / b_mn: the operand lies with its M / N axis contiguous instead of K.
struct HlProduct {
    int tiles_m = 0, tiles_n = 0, kb = 0, splits = 1, a_mn = 0, b_mn = 0;
    __host__ __device__ int tiles() const { return tiles_m * tiles_n; }
    // row blocks fastest, HL_GROUP of them at a time: B is read once per group, whatever its size
    __device__ void at(int t, int &m, int &n) const {
        const unsigned group = (unsigned)HL_GROUP * tiles_n, g = (unsigned)t / group, in = (unsigned)t - g * group;
        const unsigned gm = min(HL_GROUP, tiles_m - (int)g * HL_GROUP);
        n = in / gm;
        m = g * HL_GROUP + in - n * gm;
    }
};
// What a pair of SMs does, one part of a tile after the other. One product (forward): every pairs-th tile. Three (backward): every pairs-th of
// [dh's parts][dW's], a product's by part of K, then by tile, and behind them its share of ds's tiles, which are short: the shares level out what
// the long parts leave uneven.
//   So the pairs that run side by side walk the same stretch of K together and what they read they share through the L2: with equal shares of
// all K blocks instead (tiles cut where a share ends) each was somewhere else, 15 of 38 million sectors missed the near L2, and the
// products took as long as with a quarter of the pairs idle in the last round.
constexpr int HL_MOST_PAIRS = 127;
struct HlTrio { HlProduct p[3]; int share[HL_MOST_PAIRS + 1]; };      // dh, dW, ds; pair q has ds's tiles share[q] .. share[q + 1] - 1
struct HlOne {
    const HlProduct &pr;
    int pairs, t;
    static constexpr int g = 0, sp = 0, k0 = 0;
    int k1;
    __device__ HlOne(const HlProduct &pr, int pair, int pairs) : pr(pr), pairs(pairs), t(pair), k1(pr.kb) {}
    __device__ __forceinline__ const HlProduct &product() const { return pr; }
    __device__ __forceinline__ bool more() const { return t < pr.tiles(); }
    __device__ __forceinline__ void next() { t += pairs; }
};
struct HlThree {
    const HlTrio &w;
    int pairs, i, end, g = 0, t = 0, sp = 0, k0 = 0, k1 = 0;
    __device__ HlThree(const HlTrio &w, int pair, int pairs) : w(w), pairs(pairs), i(pair), end(w.share[pair + 1]) { place(w.share[pair]); }
    __device__ __forceinline__ const HlProduct &product() const { return w.p[g]; }
    __device__ __forceinline__ bool more() const { return g < 2 || t < end; }
    __device__ __forceinline__ void next() {
        if (g == 2) { ++t; return; }
        i += pairs;
        place(-1);
    }
    __device__ __forceinline__ void place(int first) {
        const int n0 = w.p[0].tiles() * w.p[0].splits, n1 = w.p[1].tiles() * w.p[1].splits;
        if (i >= n0 + n1) {
            g = 2; sp = 0; k0 = 0; k1 = w.p[2].kb;
            t = first >= 0 ? first : w.share[i % pairs];               // i % pairs: the pair
            return;
        }
        g = i >= n0;
        const int in = g ? i - n0 : i, tiles = w.p[g].tiles(), kt = w.p[g].kb;
        sp = in / tiles;
        t = in - sp * tiles;
        k0 = (int)((long long)kt * sp / w.p[g].splits);
        k1 = (int)((long long)kt * (sp + 1) / w.p[g].splits);
    }
};
// The roles of the kernel. An epilogue warp takes its 32 x 64 block of a complete accumulator into registers, hands the accumulator back at once, and
// works on them while what the next tile needs of its rows (epi.fetch) is on its way.
// The K loops stay rolled: where the compiler unrolls them the forward pass takes 341 us for 292 (32768 x 8192 x 768).
// FINE: operands of three terms, a stage holds a block of all of them, and an accumulator a block's products.
template <bool FINE, class Work, class What, class Epi>
__device__ __forceinline__ void hl_body(const HlMaps &maps, const What &what, Epi &epi) {
    constexpr int TERMS = FINE ? 3 : 1, STAGE = TERMS * HL_STAGE, STAGES = HL_STAGES / TERMS, OPERAND = TERMS * HL_HALF;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;      // the same offset in both CTAs: one descriptor serves both
    uint8_t *sm = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t mb = base + HL_STAGES * HL_STAGE;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + HL_STAGES * HL_STAGE + 512);
    auto bar_full = [&](int s) { return mb + 8 * s; };                 // used in the first CTA only
    auto bar_empty = [&](int s) { return mb + 64 + 8 * s; };
    auto bar_acc_full = [&](int a) { return mb + 128 + 8 * a; };
    auto bar_acc_empty = [&](int a) { return mb + 144 + 8 * a; };      // used in the first CTA only
    const uint32_t bar_left = mb + 160;                               // used in the first CTA only, where a wait has run out
    auto bar_quarters = [&](int sub, int a) { return mb + 192 + 32 * sub + 8 * a; };   // three of a row's column quarters are in shared memory

    const int tid = threadIdx.x, lane = tid & 31, warp = warp_uniform(tid >> 5);
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (tid == 0) {
        for (int s = 0; s < HL_STAGES; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(bar_acc_full(a), 1); mbar_init(bar_acc_empty(a), 2 * HL_EPI); }
        for (int q = 0; q < 16; ++q) mbar_init(bar_quarters(q >> 2, q & 3), 3);
        mbar_init(bar_left, 1);
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

    Work w(what, pair, pairs);
    int m, n;
    if (warp == 0) {
        // ------------------------------------------------------------------------------------------ producer (both CTAs)
        const bool leader = elect_one(), dirty = epi.dirty();
        uint32_t it = 0;
        bool ok = true;
        for (; w.more() && ok; w.next()) {
            const HlProduct &p = w.product();
            p.at(w.t, m, n);
            const int m0 = m * HL_B + (int)rank * (HL_B / 2), n0 = n * HL_B + (int)rank * (HL_B / 2);
            const CUtensorMap *ma = &maps.a[w.g], *mbm = w.g == 1 && dirty ? &maps.clean : &maps.b[w.g];
#pragma unroll 1
            for (int k = w.k0; k < w.k1 && ok; ++k, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(bar_empty(s), ((it / STAGES) + 1) & 1, 91));
                if (ok && leader) {
                    const int c = k * HL_BK;
                    const uint32_t full0 = cluster_addr(bar_full(s), 0);
                    if (rank == 0) mbar_expect_tx(bar_full(s), 2 * STAGE);         // both CTAs' bytes
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t sa = base + s * STAGE + t * HL_HALF, sb = sa + OPERAND;
                        if (p.a_mn) {                                  // 64 rows of K, 64 contiguous rows of M at a time
                            lp_tma_load(sa, ma, full0, m0, c, t);
                            lp_tma_load(sa + HL_HALF / 2, ma, full0, m0 + 64, c, t);
                        } else {
                            lp_tma_load(sa, ma, full0, c, m0, t);
                        }
                        if (p.b_mn) {
                            lp_tma_load(sb, mbm, full0, n0, c, t);
                            lp_tma_load(sb + HL_HALF / 2, mbm, full0, n0 + 64, c, t);
                        } else {
                            lp_tma_load(sb, mbm, full0, c, n0, t);
                        }
                    }
                }
                __syncwarp();
            }
        }
        // Nobody leaves with copies into shared memory under way, which a wait that ran out may have left there: the stages written last, both CTAs' halves
        // (the barriers count both, and the other CTA waits for this one below). All of them have long arrived where every wait was met.
        if (rank == 0) {
            const uint32_t issued = ok ? it : it - 1;
            bool here = true;
            for (uint32_t j = issued > STAGES ? issued - STAGES : 0; j < issued && here; ++j)
                here = __all_sync(0xffffffffu, mbar_wait(bar_full(j % STAGES), (j / STAGES) & 1, 91));
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------------------------------ MMA issuer (first CTA)
        if (rank == 0) {
            uint32_t it = 0, ai = 0;                                   // blocks, accumulators so far
            bool ok = true;
            auto fresh = [&]() {                                       // the next accumulator, once it has been read
                if (ai >= 2) ok = __all_sync(0xffffffffu, lp_wait_cluster(bar_acc_empty(ai & 1), ((ai >> 1) + 1) & 1, 92));
                tc_fence_after();
                return ok;
            };
            auto done = [&]() {
                lp_commit_elect(bar_acc_full(ai & 1));
                lp_commit_elect(cluster_addr(bar_acc_full(ai & 1), 1));
                ++ai;
            };
            for (; w.more() && ok; w.next()) {
                const int amn = w.product().a_mn, bmn = w.product().b_mn;
                const uint32_t idesc = idesc_bf16(HL_B, HL_B, amn, bmn), stepa = amn ? 128 : 2, stepb = bmn ? 128 : 2;
                if (!FINE && !fresh()) break;
#pragma unroll 1
                for (int k = w.k0; k < w.k1 && ok; ++k, ++it) {
                    if (FINE && !fresh()) break;
                    const int s = it % STAGES;
                    ok = __all_sync(0xffffffffu, lp_wait_cluster(bar_full(s), (it / STAGES) & 1, 93));
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t sa = base + s * STAGE, acc = tmem + (ai & 1) * HL_B;
                    const uint64_t da = smem_desc(sa, amn ? HL_HALF / 2 : 16, 1024), db = smem_desc(sa + OPERAND, bmn ? HL_HALF / 2 : 16, 1024);
#pragma unroll
                    for (int pp = FINE ? 0 : 5; pp < 6; ++pp) {        // the operands' terms: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
                        const uint32_t ta = (0x001102 >> (4 * pp)) & 15, tb = (0x010120 >> (4 * pp)) & 15;
#pragma unroll
                        for (int q = 0; q < HL_BK / 16; ++q)
                            lp_mma_elect(acc, da + ta * (HL_HALF >> 4) + q * stepa, db + tb * (HL_HALF >> 4) + q * stepb, idesc, FINE ? pp > 0 || q > 0 : (k > w.k0) | (q > 0));
                    }
                    lp_commit_elect(bar_empty(s));                     // the stage is free in both CTAs once these MMAs have read it
                    lp_commit_elect(cluster_addr(bar_empty(s), 1));
                    if (FINE) done();
                }
                if (!FINE && ok) done();
            }
            if (!ok) {                                                 // products under way read shared memory and write tensor memory
                lp_commit_elect(bar_left);
                __all_sync(0xffffffffu, lp_wait_cluster(bar_left, 0, 93));
            }
        }
    } else {
        // ------------------------------------------------------------------------------------------ epilogue (both CTAs)
        const int sub = warp & 3, part = (warp - 2) >> 2;
        const uint32_t lane_base = (uint32_t)(32 * sub) << 16, acc_empty0 = cluster_addr(bar_acc_empty(0), 0), acc_empty1 = cluster_addr(bar_acc_empty(1), 0);
        uint8_t *stage = sm + HL_STAGES * HL_STAGE + 1024 + (warp - 2) * HL_OUT_BYTES, *shared = sm + HL_STAGES * HL_STAGE + 1024;
        const int row_in = (int)rank * (HL_B / 2) + 32 * sub, col_in = part * HL_CW;
        HlTile x;
        x.lane = lane; x.sub = sub; x.part = part;
        epi.start(tid - 64);
        uint32_t ti = 0, ai = 0;
        bool ok = w.more();
        if (ok) {
            w.product().at(w.t, m, n);
            epi.fetch(w.g, m * HL_B + row_in + lane, n * HL_B + col_in);
        }
        for (; ok; ++ti) {
            x.n = n; x.row0 = m * HL_B + row_in; x.col0 = n * HL_B + col_in; x.ti = ti;
            x.g = w.g; x.sp = w.sp;
            epi.begin(x);
            float v[2][32];
            const uint32_t tacc = tmem + lane_base + part * HL_CW;
            auto full = [&]() {
                ok = __all_sync(0xffffffffu, mbar_wait(bar_acc_full(ai & 1), (ai >> 1) & 1, 94));
                tc_fence_after();
                return ok;
            };
            auto hand_back = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) lp_arrive_cluster(ai & 1 ? acc_empty1 : acc_empty0);
                ++ai;
            };
            // a load's registers as the wait leaves them: nothing that uses them moves ahead of it
            if constexpr (FINE) {
#pragma unroll
                for (int i = 0; i < 64; ++i) v[i >> 5][i & 31] = 0.f;
#pragma unroll 1
                for (int k = w.k0; k < w.k1 && full(); ++k) {
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        float u[16];
                        tmem_ld16_nowait(tacc + (ai & 1) * HL_B + 16 * b, u);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) asm volatile("" : "+f"(u[i]));
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[b >> 1][16 * (b & 1) + i] += u[i];
                    }
                    hand_back();
                }
                if (!ok) break;
            } else {
                if (!full()) break;
                tmem_ld32_nowait(tacc + (ai & 1) * HL_B, v[0]);
                tmem_ld32_nowait(tacc + (ai & 1) * HL_B + 32, v[1]);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 64; ++i) asm volatile("" : "+f"(v[i >> 5][i & 31]));
                if (w.k0 == w.k1) {                                    // a part of K with nothing in it (fewer blocks than parts)
#pragma unroll
                    for (int i = 0; i < 64; ++i) v[i >> 5][i & 31] = 0.f;
                }
                hand_back();
            }
            w.next();
            const bool more = w.more();
            if (more) {
                w.product().at(w.t, m, n);
                epi.fetch(w.g, m * HL_B + row_in + lane, n * HL_B + col_in);
            }
            ok = epi.tile(x, v, stage, shared, bar_quarters(sub, ti & 3)) && more;
        }
        epi.end(tid - 64, lane);
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

// What a row's target distribution is read from: a word per row (target), or a teacher's entries, no id twice: lists [N][k] of (id, probability's
// bits), ids ascending, INT_MAX behind the last; marks [N][blocks of 64 words], which of a block's words they are (64 bits) and the place of the
// first of them; ent, the sum of p log p, inf for a row without an entry, NaN for one with an id out of range.
struct HlTargets {
    const long long *target; long long ignore; const int2 *lists; const uint4 *marks; const float *ent; int k, blocks;
};

// ------------------------------------------------------------------------------------------------ forward
struct HlFwd {
    HlTargets t; float a;
    float2 *ml;                                                       // [tiles_n][Np]: maximum (times a) and sum of a tile's row
    float *dot;                                                       // the targets' s: [N], or [N][k] where there are lists
    unsigned *ticket; float *stats; long long N, Np; int V;
};
template <bool LIST>
struct HlFwdEpi {
    const HlFwd &f;
    uint4 marks; long long word;                                       // of the tile fetched for: as loaded, so that nothing waits for them yet
    uint64_t bits; int place, nx;                                      // of the tile at hand: targets by column, and the first one's place; or the target
    __device__ __forceinline__ void start(int i) { if (i == 0 && blockIdx.x == 0) { *f.ticket = 0u; f.stats[0] = 0.f; f.stats[1] = 0.f; } }
    __device__ __forceinline__ bool dirty() const { return false; }
    __device__ __forceinline__ void end(int, int) {}
    __device__ __forceinline__ void fetch(int, int r, int c) {
        const bool in = r < f.N && c < f.V;
        if constexpr (LIST) {
            marks = in ? f.t.marks[(long long)r * f.t.blocks + (c >> 6)] : make_uint4(0u, 0u, 0u, 0u);
        } else {
            word = in ? f.t.target[r] : -1;
        }
    }
    __device__ __forceinline__ void begin(const HlTile &) {
        if constexpr (LIST) { bits = (uint64_t)marks.y << 32 | marks.x; place = (int)marks.z; }
        else nx = word >= 0 && word < f.V && word != f.t.ignore ? (int)word : -1;
    }
    __device__ __forceinline__ bool tile(const HlTile &x, float (&v)[2][32], uint8_t *, uint8_t *shared, uint32_t quarters) {
        float m = -INFINITY, l = 0.f;
        const int row = x.row0 + x.lane;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int c0 = x.col0 + 32 * b;
            if (c0 >= f.V) break;
            if constexpr (LIST) {
                uint32_t todo = (uint32_t)(bits >> (32 * b));
                while (__any_sync(0xffffffffu, todo != 0u)) {
                    const float s = pick32(v[b], __ffs(todo) - 1);
                    if (todo != 0u) {
                        if ((unsigned)place < (unsigned)f.t.k) f.dot[(long long)row * f.t.k + place] = s;     // marks are a caller's: never past its row
                        ++place; todo &= todo - 1u;
                    }
                }
            } else if (__any_sync(0xffffffffu, (unsigned)(nx - c0) < 32u)) {
                const float s = pick32(v[b], nx - c0);
                if ((unsigned)(nx - c0) < 32u) f.dot[row] = s;
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
        float2 *mine = reinterpret_cast<float2 *>(shared) + ((x.ti & 3) * 128 + 32 * x.sub + x.lane) * 4;
        if (x.part != 0) {
            mine[x.part] = make_float2(m, l);
            __syncwarp();
            if (x.lane == 0) mbar_arrive(quarters);
            return true;
        }
        const bool ok = mbar_wait_warp(quarters, (x.ti >> 2) & 1, 95);
        if (ok) {
#pragma unroll
            for (int q = 1; q < 4; ++q) {
                const float2 o = mine[q];
                const float top = fmaxf(m, o.x), at = top == -INFINITY ? 0.f : top;
                l = l * fast_exp2(m - at) + o.y * fast_exp2(o.x - at);
                m = top;
            }
            if (row < f.N) f.ml[(long long)x.n * f.Np + row] = make_float2(m, l);
        }
        return ok;
    }
};
template <bool LIST, bool FINE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HL_NT, 1)
head_loss_fwd_kernel(const __grid_constant__ HlMaps maps, const __grid_constant__ HlProduct pr, const __grid_constant__ HlFwd f) {
    HlFwdEpi<LIST> epi{f};
    hl_body<FINE, HlOne>(maps, pr, epi);
}

// Joins a row's tiles: 32 rows a block (a lane each), the tiles dealt out to its 8 warps, then the block's losses and live rows as one
// partial sum; the last block to finish adds the partials up in order, so the sum does not depend on who that is.
struct HlJoin {
    HlTargets t; const float2 *ml; const float *dot; float2 *L; float *row_loss, *loss, *stats; double2 *partial; unsigned *ticket;
    long long N, Np; int V, tiles; float tau, a; int reduction;       // a: as the product's epilogue had it
};
template <bool LIST>
__global__ void __launch_bounds__(256) head_loss_join_kernel(const HlJoin j) {
    __shared__ float2 part[8][32];
    __shared__ float dots[32];
    __shared__ double2 sums[8];
    __shared__ bool last;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * 32 + lane;
    float m = -INFINITY, l = 0.f;
    if (row < j.N) {
#pragma unroll 4
        for (int n = warp; n < j.tiles; n += 8) {
            const float2 o = j.ml[(long long)n * j.Np + row];
            const float top = fmaxf(m, o.x), at = top == -INFINITY ? 0.f : top;
            l = l * fast_exp2(m - at) + o.y * fast_exp2(o.x - at);
            m = top;
        }
    }
    if constexpr (LIST) {                                              // four rows a warp, the entries over its lanes
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        for (int i = lane; i < j.t.k; i += 32) {
            int2 e[4];
            float s[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {                              // rows behind the last: the last again, all loads before the first use
                const long long at = min((long long)blockIdx.x * 32 + 4 * warp + q, j.N - 1) * j.t.k + i;
                e[q] = j.t.lists[at];
                s[q] = j.dot[at];
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (e[q].x < j.V) sum[q] = fmaf(__int_as_float(e[q].y), s[q], sum[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            sum[q] = warp_sum(sum[q]);
            if (lane == 0) dots[4 * warp + q] = sum[q];
        }
    }
    part[warp][lane] = make_float2(m, l);
    __syncthreads();
    double loss = 0.0;
    bool live = false;
    if (warp == 0 && row < j.N) {
#pragma unroll
        for (int q = 1; q < 8; ++q) {
            const float2 o = part[q][lane];
            const float top = fmaxf(m, o.x), at = top == -INFINITY ? 0.f : top;
            l = l * fast_exp2(m - at) + o.y * fast_exp2(o.x - at);
            m = top;
        }
        const float lg = log2f(l), hi = m + lg;                        // hi + lo = m + lg, exactly
        const float back = hi - m, rest = (m - (hi - back)) + (lg - back), lo = rest == rest ? rest : 0.f;
        // The sum is that of 2^(a s) with a rounded, so over a, not times ln 2, a row's logarithm is the logits' own: for a word that holds all the
        // probability l tells what a s lost in rounding to m, and L / a - s is 0 to 2^-22, where ln 2 left 1.3e-8 of s.
        const double L = (double)hi + lo;
        j.L[row] = make_float2(hi, lo);
        if (LIST) {
            const float ent = j.t.ent[row];
            live = ent != INFINITY;
            loss = (double)j.tau * j.tau * ent + j.tau * (L / j.a - (double)dots[lane]);
        } else {
            const long long w = j.t.target[row];
            live = w != j.t.ignore;
            loss = live && w >= 0 && w < j.V ? L / j.a - j.dot[row] : NAN;
            if (loss < 0.0) loss = 0.0;                                // by the rounding of l
        }
        if (!live) {
            loss = 0.0;
            if (!(l > 0.f && l < INFINITY)) j.stats[1] = 1.f;          // of whichever row: the same value
        }
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
        j.stats[0] = (float)s.y;
    }
}

// ------------------------------------------------------------------------------------------------ a teacher's lists
// A warp per row: probabilities of the entries that are there (id >= 0, logit not -inf) at the temperature, in ascending order of their
// ids (a rank per entry: k comparisons each), an id that comes again added to the first, and the marks. 4096 rows, 8192 words: 10 us at k 64, 60 at 256, 795 at
// 1024, where the k^2 comparisons a row are all of it.
__global__ void __launch_bounds__(128) head_teacher_kernel(const long long *__restrict__ in_ids, const float *__restrict__ in_logits, int2 *__restrict__ lists,
                                                           uint4 *__restrict__ marks, float *__restrict__ ent, long long N, int V, int k, float inv_tau) {
    extern __shared__ __align__(16) int teacher_smem[];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kk = (k + 3) & ~3;
    const long long row = (long long)blockIdx.x * 4 + warp;
    if (row >= N) return;
    int *id = teacher_smem + kk * warp;                                // absent ones behind all others
    int2 *sorted = reinterpret_cast<int2 *>(teacher_smem + 4 * kk) + kk * warp;
    constexpr int ABSENT = 0x7fffffff;
    float top = -INFINITY;
    bool bad = false;
    int here = 0;
    for (int j = lane; j < kk; j += 32) {
        const long long i = j < k ? in_ids[row * k + j] : -1;
        const float x = j < k ? in_logits[row * k + j] * inv_tau : -INFINITY;
        const bool is = i >= 0 && x != -INFINITY;
        bad |= is && i >= V;
        id[j] = is ? (int)(i >= V ? V : i) : ABSENT;
        if (is) { top = fmaxf(top, x); ++here; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o)); here += __shfl_xor_sync(0xffffffffu, here, o); }
    bad = __any_sync(0xffffffffu, bad);
    __syncwarp();
    float sum = 0.f;
    for (int j = lane; j < k; j += 32)
        if (id[j] != ABSENT) sum += expf(in_logits[row * k + j] * inv_tau - top);
    sum = warp_sum(sum);
    const float lse = logf(sum);
    float e = 0.f;
    for (int j = lane; j < k; j += 32) {
        const int me = id[j];
        if (me == ABSENT) continue;
        const float z = in_logits[row * k + j] * inv_tau - top, q = expf(z) / sum;
        if (!(q <= 0.f)) e += q * (z - lse);                     // NaN stays
        int rank = 0;                                                  // entries of a smaller id, or of the same one and an earlier place
        for (int i = 0; i < kk; i += 4) {
            const int4 o = *reinterpret_cast<const int4 *>(id + i);
            const int below = me + (i < (j & ~3));
            rank += (o.x < below) + (o.y < below) + (o.z < below) + (o.w < below);
        }
        const int4 own = *reinterpret_cast<const int4 *>(id + (j & ~3));
        rank += (own.x == me && (j & 3) > 0) + (own.y == me && (j & 3) > 1) + (own.z == me && (j & 3) > 2);
        sorted[rank] = make_int2(me, __float_as_int(q));
    }
    __syncwarp();
    // ids that come again: the first has their probabilities, they leave the list
    bool again = false;
    for (int j = lane; j < here; j += 32) again |= j > 0 && sorted[j].x == sorted[j - 1].x;
    if (__any_sync(0xffffffffu, again)) {
        int n = 0;
        if (lane == 0)
            for (int j = 0; j < here; ++j) {
                if (n > 0 && sorted[j].x == sorted[n - 1].x) sorted[n - 1].y = __float_as_int(__int_as_float(sorted[n - 1].y) + __int_as_float(sorted[j].y));
                else sorted[n++] = sorted[j];
            }
        here = __shfl_sync(0xffffffffu, n, 0);
        __syncwarp();
    }
    for (int j = lane; j < k; j += 32) lists[row * k + j] = j < here ? sorted[j] : make_int2(0x7fffffff, 0);
    e = warp_sum(e);
    if (lane == 0) ent[row] = bad ? NAN : here > 0 ? e : INFINITY;
    // blocks without an entry, which are nearly all, then the others, each by its first entry
    const int blocks = (V + 63) / 64;
    uint4 *mine = marks + row * blocks;
    for (int b = lane; b < blocks; b += 32) mine[b] = make_uint4(0u, 0u, 0u, 0u);
    __syncwarp();
    for (int j = lane; j < here; j += 32) {
        const int v = sorted[j].x, b = v >> 6;
        if (v >= V || (j > 0 && sorted[j - 1].x >> 6 == b)) continue;
        uint64_t bits = 0;
        for (int i = j; i < here && sorted[i].x < V && sorted[i].x >> 6 == b; ++i) bits |= 1ull << (sorted[i].x & 63);
        mine[b] = make_uint4((unsigned)bits, (unsigned)(bits >> 32), (unsigned)j, 0u);
    }
}

// ------------------------------------------------------------------------------------------------ backward
struct HlProb {
    HlTargets t; const float2 *L; const float *row_weight;            // row_weight NULL: 1
    float a;
    int row_from, V, col_from, cols, rows;                            // the piece: rows and columns it begins at, how many
};
template <bool LIST, int TERMS>
struct HlProbEpi {
    const HlProb &f;
    const CUtensorMap *map;
    int row; long long word; float2 L; float weight, ent;              // of the tile fetched for
    float a_hi, a_lo, c; bool live; int nx;                           // of the tile at hand; nx: the target's column
    __device__ __forceinline__ void fetch(int r, int c) {
        row = r < f.rows && c < f.cols ? f.row_from + r : -1;
        if (row < 0) return;
        L = f.L[row];
        weight = f.row_weight ? f.row_weight[row] : 1.f;
        if (LIST) ent = f.t.ent[row]; else word = f.t.target[row];
    }
    __device__ __forceinline__ void begin(const HlTile &) {
        a_hi = -L.x; a_lo = -L.y;
        const bool bad = LIST ? ent != ent : word != f.t.ignore && (word < 0 || word >= f.V);
        live = row >= 0 && (LIST ? ent != INFINITY : word != f.t.ignore);
        c = bad ? NAN : weight;
        if (!LIST) nx = live && !bad ? (int)word : -1;
    }
    // Rounded, the block goes out by two TMA stores a term, 32 columns each, from the warp's staging: 64-byte rows, their 16-byte chunks swapped
    // as the store's 64-byte swizzle has them, so that the row-per-lane writes touch every bank once. What lies outside the piece is not written.
    __device__ __forceinline__ void tile(const HlTile &x, float (&vv)[2][32], uint8_t *stage) {
        const int lane = x.lane;
        const bool plain = __all_sync(0xffffffffu, live && c == 1.f);  // no row to weigh or to leave out
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int c0 = x.col0 + 32 * b, v0 = f.col_from + c0;
            if (c0 >= f.cols) break;
            float (&v)[32] = vv[b];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = TERMS == 3 ? fast_exp2(fmaf(v[i], f.a, a_hi) + a_lo) : fast_exp2(fmaf(v[i], f.a, a_hi));
            const bool target = !LIST && __any_sync(0xffffffffu, (unsigned)(nx - v0) < 32u);     // of some row; a teacher's are put in behind this launch
            if (TERMS == 3 && target) {                                // before the values are taken apart
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] -= i == nx - v0 ? 1.f : 0.f;
            }
            if (!plain) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = live ? c * v[i] : 0.f;
            }
#pragma unroll
            for (int term = 0; term < TERMS; ++term) {
                if (lane == 0) tma_store_source_free();
                __syncwarp();
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
                    *reinterpret_cast<uint4 *>(stage + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)) = *reinterpret_cast<uint4 *>(o);
                }
                if (TERMS == 1 && target) {                            // over what was staged for the column
                    const int at = nx - v0;
                    const float q = pick32(v, at & 31);
                    if ((unsigned)at < 32u)
                        *reinterpret_cast<__nv_bfloat16 *>(stage + lane * 64 + (((at >> 3) ^ ((lane >> 1) & 3)) << 4) + 2 * (at & 7)) = __float2bfloat16_rn(q - c);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0 && x.row0 < f.rows) tma_store_3d(map, smem_u32(stage), c0, x.row0, term);
            }
        }
    }
};

// A teacher's columns of a piece of ds, exactly: c (q - p) from the logits that the forward pass kept, over the q that the product's epilogue wrote.
// An entry per thread. (Looked for in that epilogue, the entries of 32 rows were as long as the rest of it: 64 a row in 8192 words, 87 us
// against 43 for 4096 rows.)
template <int TERMS>
__global__ void __launch_bounds__(256) head_teacher_ds_kernel(const HlProb f, const float *__restrict__ kept, __nv_bfloat16 *__restrict__ P, long long ldp,
                                                              long long term_stride) {
    pdl_wait();
    pdl_launch_dependents();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, all = (long long)f.rows * f.t.k;
    if (i >= all) return;
    const int row = (int)(i / f.t.k), full = f.row_from + row;
    const int2 e = f.t.lists[(long long)f.row_from * f.t.k + i];
    const int col = e.x - f.col_from;
    if (col < 0 || col >= f.cols) return;
    const float2 L = f.L[full];
    const float ent = f.t.ent[full], c = ent != ent ? NAN : f.row_weight ? f.row_weight[full] : 1.f;
    float x = c * (fast_exp2(fmaf(kept[(long long)f.row_from * f.t.k + i], f.a, -L.x) - L.y) - __int_as_float(e.y));
#pragma unroll
    for (int term = 0; term < TERMS; ++term) {
        const __nv_bfloat16 h = __float2bfloat16_rn(x);
        P[term * term_stride + row * ldp + col] = h;
        x -= __bfloat162float(h);
    }
}

// The upstream scale that all rows share: g the gradient of the (summed or averaged) loss, count the rows averaged over.
__device__ __forceinline__ float hl_alpha(const float *g, const float *count, float tau, int reduction) {
    if (reduction == 0) return tau;
    if (reduction == 1) return tau * *g;
    const float n = *count;
    return n > 0.f ? tau * *g / n : 0.f;                              // no row counts: no gradient (the loss itself is 0 / 0)
}
// What becomes of a product's tiles: out = alpha * (acc +) C, or acc (+)= C where further pieces follow or the other parts of K have sums of
// their own, which a kernel behind this one adds up. acc [splits][rows][d] fp32.
struct HlGrad { float *acc; void *out; long long rows; int adds, last; };
struct HlGrads { HlGrad g[2]; const float *up, *count; float tau; int reduction, d, out_f32; };
struct HlGradEpi {
    const HlGrads &f;
    const HlProduct *pr;
    float alpha;
    __device__ __forceinline__ void put(const HlGrad &o, long long at, float4 val) const {
        val.x *= alpha; val.y *= alpha; val.z *= alpha; val.w *= alpha;
        if (f.out_f32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(o.out) + at) = val;
        } else {
            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(val.x, val.y), __floats2bfloat162_rn(val.z, val.w)};
            *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(o.out) + at) = *reinterpret_cast<uint2 *>(h);
        }
    }
    __device__ __forceinline__ void tile(const HlTile &x, float (&v)[2][32], uint8_t *stage) {
        const HlGrad &o = f.g[x.g];
        const int lane = x.lane, splits = pr[x.g].splits, rl = lane >> 2, cl = 4 * (lane & 3);
        if (x.col0 >= f.d || x.row0 >= o.rows) return;
        const long long plane = o.rows * f.d, base = (long long)(x.row0 + rl) * f.d + x.col0 + cl;
        float *acc = o.acc ? o.acc + x.sp * plane + base : nullptr;
        auto chunk_at = [&](int r, int ch) { return stage + r * 64 + ((ch ^ ((r >> 1) & 3)) << 4); };
        const bool direct = o.last && splits == 1;
#pragma unroll
        for (int b = 0; b < 4; ++b) {                                  // 16 columns: through shared memory, so that rows leave in 64-byte pieces
            const bool in_cols = x.col0 + 16 * b + cl < f.d;
            float4 old[4];
            if (direct && o.adds) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    old[q] = in_cols && x.row0 + rl + 8 * q < o.rows ? *reinterpret_cast<const float4 *>(acc + 8LL * q * f.d + 16 * b) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
                const float *s = &v[b >> 1][16 * (b & 1) + 4 * ch];
                *reinterpret_cast<float4 *>(chunk_at(lane, ch)) = make_float4(s[0], s[1], s[2], s[3]);
            }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float4 val = *reinterpret_cast<const float4 *>(chunk_at(rl + 8 * q, lane & 3));
                if (in_cols && x.row0 + rl + 8 * q < o.rows) {
                    float *to = acc + 8LL * q * f.d + 16 * b;
                    if (direct) {
                        if (o.adds) { val.x += old[q].x; val.y += old[q].y; val.z += old[q].z; val.w += old[q].w; }
                        put(o, base + 8LL * q * f.d + 16 * b, val);
                    } else if (o.adds) {                               // nobody else adds to it in this launch, so the order is that of the pieces
                        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(to), "f"(val.x), "f"(val.y), "f"(val.z), "f"(val.w) : "memory");
                    } else {
                        *reinterpret_cast<float4 *>(to) = val;
                    }
                }
            }
            __syncwarp();
        }
    }
};
// out = alpha * the sum over the parts of K, in their order; four columns a thread
__global__ void __launch_bounds__(256) head_loss_sum_kernel(const float *__restrict__ acc, void *__restrict__ out, long long n, int splits, const float *up,
                                                            const float *count, float tau, int reduction, int out_f32) {
    pdl_wait();
    pdl_launch_dependents();
    const float alpha = hl_alpha(up, count, tau, reduction);
    for (long long i = 4 * ((long long)blockIdx.x * 256 + threadIdx.x); i < n; i += 1024LL * gridDim.x) {
        float4 s = *reinterpret_cast<const float4 *>(acc + i);
#pragma unroll 8
        for (int q = 1; q < splits; ++q) {
            const float4 o = *reinterpret_cast<const float4 *>(acc + q * n + i);
            s.x += o.x; s.y += o.y; s.z += o.z; s.w += o.w;
        }
        s.x *= alpha; s.y *= alpha; s.z *= alpha; s.w *= alpha;
        if (out_f32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(out) + i) = s;
        } else {
            __nv_bfloat162 h[2] = {__floats2bfloat162_rn(s.x, s.y), __floats2bfloat162_rn(s.z, s.w)};
            *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(out) + i) = *reinterpret_cast<uint2 *>(h);
        }
    }
}
// One launch of the backward pass: the gradients' products of one piece and ds of the next, which do not depend on one another.
// dirty: not 0 where h of a row that does not count holds what is no number; the first launch then writes the clean copy (bf16; NULL: h is a copy already).
struct HlBwd { HlProb ds; HlGrads grads; const float *dirty; const __nv_bfloat16 *h; __nv_bfloat16 *clean; long long N; };
// whether a row counts
__device__ __forceinline__ bool hl_counts(const HlTargets &t, long long row) { return t.lists ? t.ent[row] != INFINITY : t.target[row] != t.ignore; }
// by the epilogue warps of the whole grid, a warp a row (i: the thread's number among its CTA's)
__device__ __noinline__ void hl_clean(const HlBwd &f, int i) {
    const int d = f.grads.d;
    for (long long row = (i >> 5) + (long long)blockIdx.x * HL_EPI; row < f.N; row += (long long)gridDim.x * HL_EPI) {
        const bool counts = hl_counts(f.ds.t, row);
        for (int c = 8 * (i & 31); c < d; c += 256)
            *reinterpret_cast<uint4 *>(f.clean + row * d + c) = counts ? *reinterpret_cast<const uint4 *>(f.h + row * d + c) : make_uint4(0u, 0u, 0u, 0u);
    }
}
template <bool LIST, int TERMS>
struct HlBwdEpi {
    HlProbEpi<LIST, TERMS> ds;
    HlGradEpi grad;
    const HlBwd &f;
    __device__ __forceinline__ void start(int) {
        grad.alpha = hl_alpha(grad.f.up, grad.f.count, grad.f.tau, grad.f.reduction);
    }
    __device__ __forceinline__ void fetch(int g, int r, int c) { if (g == 2) ds.fetch(r, c); }
    __device__ __forceinline__ void begin(const HlTile &x) { if (x.g == 2) ds.begin(x); }
    __device__ __forceinline__ bool tile(const HlTile &x, float (&v)[2][32], uint8_t *stage, uint8_t *, uint32_t) {
        if (x.g == 2) {
            ds.tile(x, v, stage);
        } else {                                                       // all of them before a warp's first of ds: the staging is free
            grad.tile(x, v, stage);
            fence_proxy_async();
        }
        return true;
    }
    __device__ __forceinline__ bool dirty() const { return TERMS == 1 && *f.dirty != 0.f; }
    // The clean copy, which the next launch reads first, behind the tiles: its time grows with N d, and ahead of them the other roles would spend it in
    // their bounded waits.
    __device__ __forceinline__ void end(int i, int lane) {
        if (lane == 0) tma_store_done();
        if (TERMS == 1 && f.clean != nullptr && *f.dirty != 0.f) hl_clean(f, i);
    }
};
template <bool LIST, int TERMS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HL_NT, 1)
head_loss_bwd_kernel(const __grid_constant__ HlMaps maps, const __grid_constant__ HlTrio work, const __grid_constant__ HlBwd f) {
    HlBwdEpi<LIST, TERMS> epi{{f.ds, &maps.ds}, {f.grads, work.p, 0.f}, f};
    hl_body<TERMS == 3, HlThree>(maps, work, epi);
}

// x as three bf16 terms, [3][n]; eight values a thread (d, the values of a row, a multiple of 8). t not NULL: zeros in the rows that do not count
template <bool ROWS>
__global__ void __launch_bounds__(256) head_split_kernel(const float *__restrict__ x, __nv_bfloat16 *__restrict__ out, long long n, int d, const HlTargets t) {
    pdl_wait();
    pdl_launch_dependents();
    for (long long i = 8 * ((long long)blockIdx.x * 256 + threadIdx.x); i < n; i += 2048LL * gridDim.x) {
        float v[8];
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x + i);
        *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(x + i + 4);
        if (ROWS && !hl_counts(t, i / d)) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = 0.f;
        }
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
// what warps store ds through: 32 x 32 blocks, 64-byte swizzle
static bool hl_store_map(CUtensorMap *m, const HlOperand &o, long long rows, long long cols) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)o.terms};
    const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.terms > 1 ? o.term_stride : rows * o.ld) * 2};
    const cuuint32_t box[3] = {32, 32, 1};
    return tc_encode_map(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, o.ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}
// rows x cols of it as K-major blocks of 128 x 64, or as 64 x 64 ones whose columns are M or N
static bool hl_map(CUtensorMap *m, const HlOperand &o, long long row_from, long long col_from, long long rows, long long cols, bool mn) {
    const char *p = static_cast<const char *>(o.ptr) + 2 * (row_from * o.ld + col_from);
    return tc_make_map(m, p, o.terms, rows, cols, o.ld, o.terms > 1 ? o.term_stride : rows * o.ld, mn ? 64 : 128);
}

struct HlFwdPlan { long long Np, tiles, off_ml, off_dot, off_partial, off_ticket, off_h, off_w, total; };
static HlFwdPlan hl_fwd_plan(long long N, int V, int d, int dtype) {
    HlFwdPlan p;
    p.Np = hl_up(N, 32); p.tiles = hl_tiles(V);
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += hl_up(bytes, 256); return o; };
    p.off_ml = take(p.tiles * p.Np * 8);
    p.off_dot = take(p.Np * 4);
    p.off_partial = take(p.Np / 32 * 16);
    p.off_ticket = take(4);
    p.off_h = dtype == PGB_F32 ? take(6 * N * d) : 0;
    p.off_w = dtype == PGB_F32 ? take(6LL * V * d) : 0;
    p.total = at;
    return p;
}
long long head_loss_fwd_bytes(long long N, int V, int d, int dtype) { return hl_fwd_plan(N, V, d, dtype).total; }

// the operand as the products take it; fp32: split into `room` first (t: without the rows that do not count)
static int hl_operand(HlOperand &o, const void *x, int dtype, long long rows, int d, void *room, cudaStream_t stream, const HlTargets *t = nullptr) {
    o = {x, 1, 0, d};
    if (dtype != PGB_F32) return PGB_OK;
    const long long n = rows * d, blocks = (n / 8 + 255) / 256;
    o = {room, 3, n, d};
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096));
    const cudaError_t e = t ? pdl_launch(head_split_kernel<true>, grid, dim3(256), 0, stream, static_cast<const float *>(x), static_cast<__nv_bfloat16 *>(room), n, d, *t)
                            : pdl_launch(head_split_kernel<false>, grid, dim3(256), 0, stream, static_cast<const float *>(x), static_cast<__nv_bfloat16 *>(room), n, d, HlTargets{});
    if (e != cudaSuccess) { set_cuda_error(e, "head_split launch"); return PGB_ERR_CUDA; }
    return check_launch("head_split_kernel");
}
static int hl_no_map() { set_cuda_error(cudaErrorUnknown, "cuTensorMapEncodeTiled"); return PGB_ERR_CUDA; }

static_assert(4 * 1024 * 12 <= 49152, "a teacher's entries in shared memory");
int head_teacher_launch(const long long *in_ids, const float *in_logits, int *lists, unsigned *marks, float *ent, long long N, int V, int k, float tau,
                        cudaStream_t stream) {
    const cudaError_t e = pdl_launch(head_teacher_kernel, dim3((unsigned)((N + 3) / 4)), dim3(128), (size_t)(4 * ((k + 3) & ~3) * 12), stream, in_ids, in_logits,
                                     reinterpret_cast<int2 *>(lists), reinterpret_cast<uint4 *>(marks), ent, N, V, k, 1.0f / tau);
    if (e != cudaSuccess) { set_cuda_error(e, "head_teacher launch"); return PGB_ERR_CUDA; }
    return check_launch("head_teacher_kernel");
}

int head_loss_fwd_launch(const HeadLossArgs &x, float *row_loss, float *loss, float *stats, float *L, void *scratch, cudaStream_t stream) {
    const bool list = x.lists != nullptr;
    const HlFwdPlan pl = hl_fwd_plan(x.N, x.V, x.d, x.dtype);
    char *s = static_cast<char *>(scratch);
    HlOperand h, w;
    int rc = hl_operand(h, x.h, x.dtype, x.N, x.d, s + pl.off_h, stream);
    if (rc == PGB_OK) rc = hl_operand(w, x.W, x.dtype, x.V, x.d, s + pl.off_w, stream);
    if (rc != PGB_OK) return rc;
    HlMaps maps;
    if (!hl_map(&maps.a[0], h, 0, 0, x.N, x.d, false) || !hl_map(&maps.b[0], w, 0, 0, x.V, x.d, false)) return hl_no_map();
    HlProduct pr;
    pr.tiles_m = hl_tiles(x.N); pr.tiles_n = (int)pl.tiles; pr.kb = (x.d + HL_BK - 1) / HL_BK;
    const HlTargets t{x.target, x.ignore, reinterpret_cast<const int2 *>(x.lists), reinterpret_cast<const uint4 *>(x.marks), x.ent, x.k, (x.V + 63) / 64};
    const HlFwd f{t, LOG2E_F / x.tau, reinterpret_cast<float2 *>(s + pl.off_ml), list ? x.kept : reinterpret_cast<float *>(s + pl.off_dot),
                  reinterpret_cast<unsigned *>(s + pl.off_ticket), stats, x.N, pl.Np, x.V};
    if (h.terms == 3)
        rc = list ? hl_launch(head_loss_fwd_kernel<true, true>, 0, "head_loss_fwd_kernel", maps, pr, pr.tiles(), f, stream)
                  : hl_launch(head_loss_fwd_kernel<false, true>, 1, "head_loss_fwd_kernel", maps, pr, pr.tiles(), f, stream);
    else
        rc = list ? hl_launch(head_loss_fwd_kernel<true, false>, 2, "head_loss_fwd_kernel", maps, pr, pr.tiles(), f, stream)
                  : hl_launch(head_loss_fwd_kernel<false, false>, 3, "head_loss_fwd_kernel", maps, pr, pr.tiles(), f, stream);
    if (rc != PGB_OK) return rc;
    const HlJoin j{t, f.ml, f.dot, reinterpret_cast<float2 *>(L), row_loss, loss, stats, reinterpret_cast<double2 *>(s + pl.off_partial), f.ticket,
                   x.N, pl.Np, x.V, (int)pl.tiles, x.tau, f.a, x.reduction};
    cudaError_t e = pdl_launch(list ? head_loss_join_kernel<true> : head_loss_join_kernel<false>, dim3((unsigned)(pl.Np / 32)), dim3(256), 0, stream, j);
    if (e != cudaSuccess) { set_cuda_error(e, "head_loss_join launch"); return PGB_ERR_CUDA; }
    return check_launch("head_loss_join_kernel");
}

// How the backward pass is cut: pieces of `step` rows (by_rows) or columns, and the parts of K of the two gradients' products.
struct HlBwdPlan {
    bool by_rows; long long step, pieces, ldp, rows, cols; int terms, s_dh[2], s_dw[2];          // parts in all pieces but the last, in the last
    long long off_p[2], off_dh, off_dw, off_h, off_w, total;
};
// A launch's work in units of the time of a K block's one product (0.33 us; np of them a block): a part of a tile costs its own and about four
// more (its epilogue's end and the next one's beginning).
struct HlLoad {
    long long n0, n, f0, r0, f, r; double c0, c1;                      // parts of the first product, of both; rounds and rest of either number over the pairs
    HlLoad(long long t0, long long k0, int s0, long long t1, long long k1, int s1, int pairs) : n0(t0 * s0), n(t0 * s0 + t1 * s1), f0(n0 / pairs), r0(n0 % pairs),
        f(n / pairs), r(n % pairs), c0((double)k0 / s0 + 4.0), c1((double)k1 / s1 + 4.0) {}
    double of(long long p) const {                                     // pair p's long parts
        const long long first = f0 + (p < r0), both = f + (p < r);
        return first * c0 + (both - first) * c1;
    }
    double most() const {                                              // of the first pair, or of the first behind the last full round of either product
        const double a = of(0), b = of(r0), c = of(r);
        return a > b ? (a > c ? a : c) : (b > c ? b : c);
    }
    double all() const { return n0 * c0 + (n - n0) * c1; }
};
constexpr double HL_DS = 5.0;                                         // what a tile of ds costs beyond its K blocks
constexpr int HL_LONGEST = 4096;                                      // blocks of a part, 1.4 ms of products: an epilogue's wait for one is bounded by milliseconds
struct HlSplits { int dh, dw; double cost; };
// The parts of K with which the pairs finish earliest, `filler` units of short tiles dealt out behind them. fix0, fix1: parts that are given (0: to be chosen).
static HlSplits hl_splits(long long t0, long long k0, long long t1, long long k1, double filler, int np, int pairs, int fix0, int fix1) {
    static const int choice[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32};
    HlSplits best{1, 1, 1e300};
    for (int a : choice) {
        if (a > 1 && (fix0 || t0 == 0 || k0 / a < 4 * np)) break;
        if (np == 1 && t0 > 0 && !fix0 && k0 > (long long)HL_LONGEST * a) continue;              // three terms: an accumulator is a block's
        for (int b : choice) {
            if (b > 1 && (fix1 || t1 == 0 || k1 / b < 4 * np)) break;
            if (np == 1 && t1 > 0 && !fix1 && k1 > (long long)HL_LONGEST * b) continue;
            const int s0 = fix0 ? fix0 : a, s1 = fix1 ? fix1 : b;
            const HlLoad load(t0, k0, s0, t1, k1, s1, pairs);
            const double level = (load.all() + filler) / pairs, most = load.most();
            // the kernel that adds up the parts' sums: 10 and what it reads, 256 KiB a tile and part
            const double cost = (level > most ? level : most) + (s0 > 1 ? 10.0 + 0.15 * t0 * s0 : 0.0) + (s1 > 1 ? 10.0 + 0.15 * t1 * s1 : 0.0);
            if (cost < best.cost) best = {s0, s1, cost};
        }
    }
    return best;
}
static HlBwdPlan hl_bwd_plan(long long N, int V, int d, int dtype, bool dh, bool dw) {
    HlBwdPlan p;
    p.terms = dtype == PGB_F32 ? 3 : 1;
    p.by_rows = N >= V;
    const int pairs = sm_count() / 2, np = p.terms == 3 ? 6 : 1;
    const long long most = HL_PIECE_BYTES / (2 * p.terms), across = hl_up(p.by_rows ? V : N, 64), along = p.by_rows ? N : V;
    const long long td = hl_tiles(d), kd = (d + HL_BK - 1) / HL_BK * np, ta = hl_tiles(across), ka = (across + HL_BK - 1) / HL_BK * np;
    const bool along_d = p.by_rows ? dh : dw, across_d = p.by_rows ? dw : dh;                    // the gradient that has a piece's rows, the one that gathers over pieces
    // a launch with the products of n rows or columns and ds of the next m
    auto of = [&](long long n, long long m, int gather) {
        const long long t0 = along_d ? hl_tiles(n) * td : 0, t1 = across_d ? ta * td : 0, k1 = (n + HL_BK - 1) / HL_BK * np;
        const double filler = (double)hl_tiles(m) * ta * (kd + HL_DS);
        HlSplits s = p.by_rows ? hl_splits(t0, ka, t1, k1, filler, np, pairs, 0, gather) : hl_splits(t1, k1, t0, ka, filler, np, pairs, gather, 0);
        s.cost += 20.0;                                                // a launch's beginning and end
        return s;
    };
    long long step = most / across / HL_B * HL_B;
    if (step < HL_B) step = HL_B;
    HlSplits best{1, 1, 1e300}, last{1, 1, 0.0};
    if (step >= along) {
        p.step = hl_up(along, HL_B);
        best = last = of(along, 0, 0);
    } else {
        const long long stride = step / 32 / HL_B * HL_B + HL_B;       // sixteen steps or fewer are looked at
        for (long long n = step; 2 * n > step; n -= stride) {          // the one whose launches take the least
            const long long pieces = (along + n - 1) / n, rest = along - (pieces - 1) * n;
            HlSplits s = of(n, n, 0);
            const HlSplits r = of(rest, 0, p.by_rows ? s.dw : s.dh);   // the gathering gradient's sums go on in the same parts
            s.cost = s.cost * (pieces - 1) + r.cost;
            if (s.cost < best.cost) { best = s; last = r; p.step = n; }
        }
    }
    p.pieces = (along + p.step - 1) / p.step;
    p.s_dh[0] = best.dh; p.s_dw[0] = best.dw; p.s_dh[1] = last.dh; p.s_dw[1] = last.dw;
    p.ldp = p.by_rows ? hl_up(V, 64) : p.step;
    p.rows = p.by_rows && p.step < N ? p.step : N;
    p.cols = !p.by_rows && p.step < V ? p.step : V;
    long long at = 0;
    auto take = [&](long long bytes) { const long long o = at; at += hl_up(bytes, 256); return o; };
    p.off_p[0] = take(2 * p.terms * p.rows * p.ldp);
    p.off_p[1] = p.pieces > 1 ? take(2 * p.terms * p.rows * p.ldp) : p.off_p[0];
    // fp32 sums: of the gradient that gathers over pieces, and of one whose K axis is in parts
    const int sh = p.s_dh[0] > p.s_dh[1] ? p.s_dh[0] : p.s_dh[1], sw = p.s_dw[0] > p.s_dw[1] ? p.s_dw[0] : p.s_dw[1];
    p.off_dh = dh && (sh > 1 || (!p.by_rows && p.pieces > 1)) ? take(4LL * sh * p.rows * d) : -1;
    p.off_dw = dw && (sw > 1 || (p.by_rows && p.pieces > 1)) ? take(4LL * sw * p.cols * d) : -1;
    p.off_h = dtype == PGB_F32 ? take(6 * N * d) : dw ? take(2 * N * d) : 0;                    // its terms, or room for a clean copy
    p.off_w = dtype == PGB_F32 ? take(6LL * V * d) : 0;
    p.total = at;
    return p;
}
// pair q's tiles of ds: as many as bring it to the level that all of them reach
static void hl_share(HlTrio &w, int np, int pairs) {
    const HlProduct &a = w.p[0], &b = w.p[1];
    const int tiles = w.p[2].tiles();
    const HlLoad load(a.tiles(), (long long)a.kb * np, a.splits, b.tiles(), (long long)b.kb * np, b.splits, pairs);
    const double c = w.p[2].kb * np + HL_DS;
    double level = (load.all() + tiles * c) / pairs;
    for (int round = 0; round < 4 && load.n > 0 && tiles > 0; ++round) {                         // pairs above the level have none and raise it for the others
        double over = 0.0;
        int below = 0;
        for (int q = 0; q < pairs; ++q) {
            const double l = load.of(q);
            if (l >= level) over += l; else ++below;
        }
        if (below == 0 || below == pairs) break;
        level = (load.all() + tiles * c - over) / below;
    }
    double due = 0.0;
    for (int q = 0; q < pairs; ++q) {
        w.share[q] = (int)due < tiles ? (int)due : tiles;
        const double l = load.of(q);
        if (l < level) due += (level - l) / c;
    }
    w.share[pairs] = tiles;
}
long long head_loss_bwd_bytes(long long N, int V, int d, int dtype, int want_dh, int want_dw) {
    return hl_bwd_plan(N, V, d, dtype, want_dh != 0, want_dw != 0).total;
}
static int hl_sum(const float *acc, void *out, long long n, int splits, const HlGrads &f, cudaStream_t stream) {
    const long long blocks = (n / 4 + 255) / 256;
    cudaError_t e = pdl_launch(head_loss_sum_kernel, dim3((unsigned)(blocks < 2368 ? blocks : 2368)), dim3(256), 0, stream, acc, out, n, splits, f.up, f.count, f.tau,
                               f.reduction, f.out_f32);
    if (e != cudaSuccess) { set_cuda_error(e, "head_loss_sum launch"); return PGB_ERR_CUDA; }
    return check_launch("head_loss_sum_kernel");
}
int head_loss_bwd_launch(const HeadLossArgs &x, const float *L, const float *stats, const float *up, void *dh, void *dw, void *scratch, cudaStream_t stream) {
    const bool list = x.lists != nullptr;
    const HlBwdPlan pl = hl_bwd_plan(x.N, x.V, x.d, x.dtype, dh != nullptr, dw != nullptr);
    char *s = static_cast<char *>(scratch);
    HlOperand h, w;
    const HlTargets targets{x.target, x.ignore, reinterpret_cast<const int2 *>(x.lists), reinterpret_cast<const uint4 *>(x.marks), x.ent, x.k, (x.V + 63) / 64};
    int rc = hl_operand(h, x.h, x.dtype, x.N, x.d, s + pl.off_h, stream, &targets);
    if (rc == PGB_OK) rc = hl_operand(w, x.W, x.dtype, x.V, x.d, s + pl.off_w, stream);
    if (rc != PGB_OK) return rc;
    const int np = pl.terms == 3 ? 6 : 1, esize = x.dtype == PGB_F32 ? 4 : 2;
    const int which = (pl.terms == 3) * 2 + list;
    const int room = which == 0 ? hl_pairs(head_loss_bwd_kernel<false, 1>, 4) : which == 1 ? hl_pairs(head_loss_bwd_kernel<true, 1>, 5)
                   : which == 2 ? hl_pairs(head_loss_bwd_kernel<false, 3>, 6) : hl_pairs(head_loss_bwd_kernel<true, 3>, 7);
    if (room < 1) { set_cuda_error(cudaGetLastError(), "head_loss_bwd_kernel"); return PGB_ERR_CUDA; }
    auto at = [&](long long off) { return off >= 0 ? reinterpret_cast<float *>(s + off) : nullptr; };
    auto piece = [&](int i) { return HlOperand{s + pl.off_p[i & 1], pl.terms, pl.rows * pl.ldp, pl.ldp}; };
    HlBwd f{};
    f.ds.t = targets;
    f.ds.L = reinterpret_cast<const float2 *>(L); f.ds.row_weight = x.reduction == 0 ? up : nullptr; f.ds.a = LOG2E_F / x.tau; f.ds.V = x.V;
    f.grads.up = up; f.grads.count = stats; f.grads.tau = x.tau; f.grads.reduction = x.reduction; f.grads.d = x.d; f.grads.out_f32 = x.dtype == PGB_F32;
    const HlOperand clean{s + pl.off_h, 1, 0, x.d};                    // bf16: filled by the first launch where it is needed
    f.dirty = stats + 1; f.h = static_cast<const __nv_bfloat16 *>(x.h); f.N = x.N;
    // launch i: the products of piece i - 1, ds of piece i
    for (long long i = 0; i <= pl.pieces; ++i) {
        HlMaps maps;
        HlTrio work{};
        f.clean = i == 0 && dw && pl.terms == 1 ? static_cast<__nv_bfloat16 *>(const_cast<void *>(clean.ptr)) : nullptr;
        auto rows_of = [&](long long j) { return pl.by_rows && (j + 1) * pl.step > x.N ? x.N - j * pl.step : pl.rows; };
        auto cols_of = [&](long long j) { return !pl.by_rows && (j + 1) * pl.step > x.V ? x.V - j * pl.step : pl.cols; };
        bool mapped = true;
        if (i < pl.pieces) {
            const long long rows = rows_of(i), cols = cols_of(i), row_from = pl.by_rows ? i * pl.step : 0, col_from = pl.by_rows ? 0 : i * pl.step;
            mapped = hl_map(&maps.a[2], h, row_from, 0, rows, x.d, false) && hl_map(&maps.b[2], w, col_from, 0, cols, x.d, false) && hl_store_map(&maps.ds, piece(i), rows, cols);
            HlProduct &q = work.p[2];
            q.tiles_m = hl_tiles(rows); q.tiles_n = hl_tiles(cols); q.kb = (x.d + HL_BK - 1) / HL_BK;
            f.ds.row_from = (int)row_from; f.ds.rows = (int)rows; f.ds.col_from = (int)col_from; f.ds.cols = (int)cols;
        }
        if (i > 0) {
            const long long j = i - 1, rows = rows_of(j), cols = cols_of(j), row_from = pl.by_rows ? j * pl.step : 0, col_from = pl.by_rows ? 0 : j * pl.step;
            const bool first = j == 0, last = i == pl.pieces;
            if (dh) {                                                  // dh[rows] += ds W[cols]
                mapped = mapped && hl_map(&maps.a[0], piece(j), 0, 0, rows, cols, false) && hl_map(&maps.b[0], w, col_from, 0, cols, x.d, true);
                HlProduct &q = work.p[0];
                q.tiles_m = hl_tiles(rows); q.tiles_n = hl_tiles(x.d); q.kb = (int)((cols + HL_BK - 1) / HL_BK); q.splits = pl.s_dh[last]; q.b_mn = 1;
                const bool gathers = !pl.by_rows && pl.pieces > 1;
                f.grads.g[0] = {at(pl.off_dh), static_cast<char *>(dh) + row_from * x.d * esize, rows, gathers && !first, !gathers || last};
            }
            if (dw) {                                                  // dW[cols] += ds^T h[rows]
                mapped = mapped && hl_map(&maps.a[1], piece(j), 0, 0, rows, cols, true) && hl_map(&maps.b[1], h, row_from, 0, rows, x.d, true) &&
                         (pl.terms == 3 || hl_map(&maps.clean, clean, row_from, 0, rows, x.d, true));
                HlProduct &q = work.p[1];
                q.tiles_m = hl_tiles(cols); q.tiles_n = hl_tiles(x.d); q.kb = (int)((rows + HL_BK - 1) / HL_BK); q.splits = pl.s_dw[last]; q.a_mn = 1; q.b_mn = 1;
                const bool gathers = pl.by_rows && pl.pieces > 1;
                f.grads.g[1] = {at(pl.off_dw), static_cast<char *>(dw) + col_from * x.d * esize, cols, gathers && !first, !gathers || last};
            }
        }
        if (!mapped) return hl_no_map();
        const long long parts = (long long)work.p[0].tiles() * work.p[0].splits + (long long)work.p[1].tiles() * work.p[1].splits + work.p[2].tiles();
        const int pairs = (int)(parts < room ? parts : room < HL_MOST_PAIRS ? room : HL_MOST_PAIRS);
        hl_share(work, np, pairs);
        rc = which == 0 ? hl_launch(head_loss_bwd_kernel<false, 1>, 4, "head_loss_bwd_kernel", maps, work, pairs, f, stream)
           : which == 1 ? hl_launch(head_loss_bwd_kernel<true, 1>, 5, "head_loss_bwd_kernel", maps, work, pairs, f, stream)
           : which == 2 ? hl_launch(head_loss_bwd_kernel<false, 3>, 6, "head_loss_bwd_kernel", maps, work, pairs, f, stream)
                        : hl_launch(head_loss_bwd_kernel<true, 3>, 7, "head_loss_bwd_kernel", maps, work, pairs, f, stream);
        if (rc == PGB_OK && list && i < pl.pieces) {
            const HlOperand P = piece(i);
            __nv_bfloat16 *to = static_cast<__nv_bfloat16 *>(const_cast<void *>(P.ptr));
            const dim3 grid((unsigned)(((long long)f.ds.rows * x.k + 255) / 256));
            const cudaError_t e = pl.terms == 3 ? pdl_launch(head_teacher_ds_kernel<3>, grid, dim3(256), 0, stream, f.ds, (const float *)x.kept, to, P.ld, P.term_stride)
                                                : pdl_launch(head_teacher_ds_kernel<1>, grid, dim3(256), 0, stream, f.ds, (const float *)x.kept, to, P.ld, P.term_stride);
            if (e != cudaSuccess) { set_cuda_error(e, "head_teacher_ds launch"); return PGB_ERR_CUDA; }
        }
        for (int g = 0; g < 2 && rc == PGB_OK && i > 0; ++g) {
            const HlGrad &o = f.grads.g[g];
            if (work.p[g].tiles() > 0 && work.p[g].splits > 1 && o.last) rc = hl_sum(o.acc, o.out, o.rows * x.d, work.p[g].splits, f.grads, stream);
        }
        if (rc != PGB_OK) return rc;
    }
    return PGB_OK;
}

int head_loss_error_flag(int *out) { return tc_read_error_flag(out); }

}  // namespace pgb
