// Embedding lookup with scaling, y_n = scale w_{id_n}, and its gradient dw_v = scale sum_{n: id_n = v} g_n by sorted tokens: no atomics on
// the sums, so the same call gives the same bits, and a word's gradients are added in fp32 and rounded once.
//   Both directions move bytes and compute nothing to speak of: the lookup reads and writes N rows, the gradient reads N rows and writes V.
//   The gradient of more than EB_FEW tokens is three launches, each a programmatic dependent of the one before (32768 tokens of a text, 8192 words of
//   768 bf16, alone with cold caches: 13 + 14 + 12 us, of which the bytes are 10; the lookup 12 for 10):
//   embed_sort_kernel  a CTA owns a share of the vocabulary and reads all ids once (8 N bytes from the L2), which tells it its own tokens
//                      in order and how many belong to the CTAs before it: a stable counting sort without a word exchanged between CTAs.
//   embed_sum_kernel   the sorted tokens in chunks of EB_CHUNK, whatever words they hold, so a frequent word is spread over many CTAs: a run
//                      that lies in one chunk is finished there, one that crosses a border leaves fp32 partial sums. Further CTAs write the
//                      zeros of words that no token has.
//   embed_join_kernel  adds the partial sums of the runs that cross borders, in order.
#include "common.cuh"

namespace pgb {

constexpr int EB_WARPS = 32, EB_NT = EB_WARPS * 32, EB_ROWS = 512, EB_LIST = 128;  // sort: warps, most words a CTA owns, a warp's list of its tokens
constexpr int EB_LOADS = 16;                                          // ids that a lane has on their way
constexpr int EB_CHUNK = 32, EB_ZERO = 32;                            // sorted tokens of a summing CTA, words of a zeroing one

// 16 bytes of T, or one element where a row is no whole number of them; Raw: as loaded
template <typename T, int VEC> struct EbPack;
template <typename T> struct EbPack<T, 1> {
    using Raw = T;
    static __device__ __forceinline__ Raw load(const T *p) { return *p; }
    static __device__ __forceinline__ void floats(Raw r, float (&v)[1]) { v[0] = to_f32(r); }
    static __device__ __forceinline__ void store(T *p, const float (&v)[1]) { from_f32(*p, v[0]); }
};
template <> struct EbPack<float, 4> {
    using Raw = float4;
    static __device__ __forceinline__ Raw load(const float *p) { return *reinterpret_cast<const float4 *>(p); }
    static __device__ __forceinline__ void floats(Raw r, float (&v)[4]) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
    static __device__ __forceinline__ void store(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
template <> struct EbPack<__nv_bfloat16, 8> {
    using Raw = uint4;
    static __device__ __forceinline__ Raw load(const __nv_bfloat16 *p) { return *reinterpret_cast<const uint4 *>(p); }
    static __device__ __forceinline__ void floats(Raw r, float (&v)[8]) {
        const uint32_t x[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(x[i] << 16); v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[8]) {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(h);
    }
};

// a warp per row; an id outside the table gives a row of NaN
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const long long *__restrict__ ids, const T *__restrict__ W, float scale, T *__restrict__ y, long long N,
                                                        int V, int d) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= N) return;
    const long long id = ids[row];
    const bool in = id >= 0 && id < V;
    const T *w = W + (in ? id : 0) * d;
    T *out = y + row * d;
#pragma unroll 4
    for (int c = lane * VEC; c < d; c += 32 * VEC) {
        float v[VEC];
        EbPack<T, VEC>::floats(EbPack<T, VEC>::load(w + c), v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = in ? scale * v[i] : __int_as_float(0x7fffffff);
        EbPack<T, VEC>::store(out + c, v);
    }
}

// ------------------------------------------------------------------------------------------------ gradient: the tokens in order of their words
// CTA b owns the words v with v mod CTAS == b (CTAS a power of two): vocabularies are numbered by frequency, and with a contiguous range each
// the CTA of the first words had a third of a text's tokens (28 us of sorting; 32768 tokens, 8192 words).
// order [N]: (token, its word), by (v mod CTAS, v), the tokens ascending within a word; run [V]: where a word's tokens begin and end there;
// run [V] (the last): how many there are. Tokens whose id is outside the table or the padding word are left out.
__global__ void __launch_bounds__(EB_NT, 1) embed_sort_kernel(const long long *__restrict__ ids, int2 *__restrict__ order, int2 *__restrict__ run, int N, int V,
                                                              long long padding, int rows_per, int log_ctas) {
    extern __shared__ int eb_smem[];
    int *hist = eb_smem;                                               // [warps][rows_per]: a warp's tokens of a word, then where its next one goes
    int2 *list = reinterpret_cast<int2 *>(hist + EB_WARPS * rows_per);
    __shared__ int below[EB_WARPS], scan[EB_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned mask = (1u << log_ctas) - 1u, b = blockIdx.x;
    const int rows = (int)b < V ? (int)((unsigned)(V - 1) - b >> log_ctas) + 1 : 0;   // words b, b + CTAS, ...
    for (int i = threadIdx.x; i < EB_WARPS * rows_per; i += EB_NT) hist[i] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    // a warp reads a contiguous share of the ids, 32 at a time, EB_LOADS loads in flight
    const int share = ((N + EB_WARPS - 1) / EB_WARPS + 31) & ~31, from = min(N, warp * share), to = min(N, from + share);
    const unsigned lt = (1u << lane) - 1u;
    int2 *mine = list + warp * EB_LIST;
    int n_below = 0, n_found = 0;
    // the id as an unsigned 32-bit number, past every word where it is none of the table or the padding: the comparisons of 64-bit ids were 125 instructions per 32
    const unsigned u_pad = padding >= 0 && padding < V ? (unsigned)padding : ~0u, words = V;
    auto visit = [&](auto &&take) {
        for (int n0 = from; n0 < to; n0 += 32 * EB_LOADS) {
            uint2 id[EB_LOADS];
            const uint2 *at = reinterpret_cast<const uint2 *>(ids) + n0 + lane;
            const bool all = n0 + 32 * EB_LOADS <= to;
#pragma unroll
            for (int j = 0; j < EB_LOADS; ++j) id[j] = all || n0 + 32 * j + lane < to ? at[32 * j] : make_uint2(0u, 1u);
#pragma unroll
            for (int j = 0; j < EB_LOADS; ++j) {
                const unsigned x = id[j].x, owner = x & mask;
                const bool use = id[j].y == 0u && x < words && x != u_pad;
                take(n0 + 32 * j + lane, (int)(x >> log_ctas), use && owner == b, use && owner < b);
            }
        }
    };
    visit([&](int n, int r, bool here, bool lower) {
        n_below += lower;
        const unsigned who = __ballot_sync(0xffffffffu, here);
        if (who == 0u) return;
        if (here) {
            const int at = n_found + __popc(who & lt);
            if (at < EB_LIST) mine[at] = make_int2(n, r);
            atomicAdd(&hist[warp * rows_per + r], 1);
        }
        n_found += __popc(who);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n_below += __shfl_xor_sync(0xffffffffu, n_below, o);
    if (lane == 0) below[warp] = n_below;
    __syncthreads();
    // a word per thread: its tokens over the warps, an exclusive scan over the words, the place of every warp's first one
    int total = 0;
    const int r0 = threadIdx.x;
    if (r0 < rows)
#pragma unroll 8
        for (int w = 0; w < EB_WARPS; ++w) total += hist[w * rows_per + r0];
    int inc = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += up; }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll 8
    for (int w = 0; w < EB_WARPS; ++w) { base += below[w]; all += scan[w]; if (w < warp) base += scan[w]; }
    if (b == mask && threadIdx.x == 0) run[V] = make_int2(base + all, 0);   // warp 0's base: everything below
    int at = base + inc - total;
    if (r0 < rows) {
        run[b + ((unsigned)r0 << log_ctas)] = make_int2(at, at + total);
#pragma unroll 8
        for (int w = 0; w < EB_WARPS; ++w) { const int c = hist[w * rows_per + r0]; hist[w * rows_per + r0] = at; at += c; }
    }
    __syncthreads();
    // a warp puts its tokens down in order: 32 at a time, the ones of a word ranked by the lanes before
    int *next = hist + warp * rows_per;
    auto put = [&](int n, int r, bool here) {
        const unsigned who = __ballot_sync(0xffffffffu, here);
        if (here) {
            const unsigned same = __match_any_sync(who, r);
            const int start = next[r];
            order[start + __popc(same & lt)] = make_int2(n, (int)(b + ((unsigned)r << log_ctas)));
            __syncwarp(who);
            if ((same & lt) == 0u) next[r] = start + __popc(same);
        }
        __syncwarp();
    };
    if (n_found <= EB_LIST) {
        for (int i = 0; i < n_found; i += 32) {
            const bool here = i + lane < n_found;
            const int2 e = here ? mine[i + lane] : make_int2(0, 0);
            put(e.x, e.y, here);
        }
    } else {                                                           // more than its list holds: the ids once more
        visit([&](int n, int r, bool here, bool) { if (__any_sync(0xffffffffu, here)) put(n, r, here); });
    }
}

// ------------------------------------------------------------------------------------------------ gradient: sums of runs
// part [chunks][2][d] fp32: 0 what a chunk adds to the run it begins inside of, 1 what it holds of the run it ends inside of
enum { EB_GOES_ON = 0, EB_WHOLE = 1, EB_HEAD = 2, EB_TAIL = 3 };      // at a token: its run has further ones here; ends, and lies here; ends, and is a part
template <typename T, int VEC>
__global__ void embed_sum_kernel(const T *__restrict__ g, const int2 *__restrict__ order, const int2 *__restrict__ run, float scale, T *__restrict__ dW,
                                 float *__restrict__ part, int chunks, int V, int d) {
    __shared__ int tok[EB_CHUNK], word[EB_CHUNK], what[EB_CHUNK];
    pdl_wait();
    pdl_launch_dependents();
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    if ((int)blockIdx.x >= chunks) {                                   // words without a token
        const int v0 = (blockIdx.x - chunks) * EB_ZERO, lane = threadIdx.x & 31;
        const int2 r = v0 + lane < V ? run[v0 + lane] : make_int2(0, 1);
        const bool none = r.x == r.y;
        unsigned todo = __ballot_sync(0xffffffffu, none);
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 0.f;
        if (c < d)
            for (; todo != 0u; todo &= todo - 1u) EbPack<T, VEC>::store(dW + (long long)(v0 + __ffs(todo) - 1) * d + c, v);
        return;
    }
    const int a = blockIdx.x * EB_CHUNK, total = run[V].x, b = min(a + EB_CHUNK, total), n = b - a;
    if (n <= 0) return;
    if ((int)threadIdx.x < n) {                                        // a token each; the block has 32 threads at least
        const int i = threadIdx.x;
        const int2 t = order[a + i];
        const bool ends = i + 1 == n || order[a + i + 1].y != t.y;
        const int2 r = ends ? run[t.y] : make_int2(0, 0);
        tok[i] = t.x;
        word[i] = t.y;
        what[i] = !ends ? EB_GOES_ON : r.x >= a && r.y <= b ? EB_WHOLE : r.x >= a ? EB_TAIL : EB_HEAD;
    }
    __syncthreads();
    if (c >= d) return;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    constexpr int AHEAD = 8;
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
        typename EbPack<T, VEC>::Raw buf[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) buf[j] = EbPack<T, VEC>::load(g + (long long)tok[min(i0 + j, n - 1)] * d + c);   // all of them before the first is used
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j;
            if (i >= n) break;
            float v[VEC];
            EbPack<T, VEC>::floats(buf[j], v);
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += v[q];
            const int w = what[i];
            if (w == EB_GOES_ON) continue;
            if (w == EB_WHOLE) {
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] *= scale;
                EbPack<T, VEC>::store(dW + (long long)word[i] * d + c, acc);
            } else {
                float *p = part + ((long long)blockIdx.x * 2 + (w == EB_TAIL)) * d + c;
#pragma unroll
                for (int q = 0; q < VEC; ++q) p[q] = acc[q];
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
        }
    }
}
// The run that begins in this chunk and goes on behind it: its partial sums, dealt out to EB_SLICES threads a column and added up in
// order. A frequent word has many (a twentieth of 32768 tokens: 51), one thread's loads one behind the other would be what the kernel takes.
constexpr int EB_SLICES = 8, EB_COLS = 64;
template <typename T, int VEC>
__global__ void __launch_bounds__(EB_SLICES * EB_COLS) embed_join_kernel(const int2 *__restrict__ order, const int2 *__restrict__ run, const float *__restrict__ part,
                                                                         float scale, T *__restrict__ dW, int V, int d) {
    __shared__ float sums[EB_SLICES][EB_COLS * 4];
    constexpr int W = VEC == 1 ? 1 : 4;                                // columns of a thread
    pdl_wait();
    pdl_launch_dependents();
    const int end = (blockIdx.x + 1) * EB_CHUNK;
    const int total = run[V].x, w = order[end].y, before = order[end - 1].y;
    if (end >= total || before != w) return;                           // no run crosses this border
    const int2 r = run[w];
    const int last = (r.y - 1) / EB_CHUNK;
    if (r.x < end - EB_CHUNK) return;                                 // it began further ahead
    const int col = threadIdx.x % EB_COLS, slice = threadIdx.x / EB_COLS, c = (blockIdx.y * EB_COLS + col) * W;
    float acc[W];
#pragma unroll
    for (int q = 0; q < W; ++q) acc[q] = 0.f;
    if (c < d) {
#pragma unroll 8
        for (int j = blockIdx.x + slice; j <= last; j += EB_SLICES) {
            const float *o = part + ((long long)j * 2 + (j == (int)blockIdx.x)) * d + c;
            float v[W];
            if constexpr (W == 4) EbPack<float, 4>::floats(EbPack<float, 4>::load(o), v); else v[0] = *o;
#pragma unroll
            for (int q = 0; q < W; ++q) acc[q] += v[q];
        }
    }
#pragma unroll
    for (int q = 0; q < W; ++q) sums[slice][col * W + q] = acc[q];
    __syncthreads();
    for (int i = threadIdx.x; i < EB_COLS * W; i += EB_SLICES * EB_COLS) {
        const int at = blockIdx.y * EB_COLS * W + i;
        if (at >= d) continue;
        float s = sums[0][i];
#pragma unroll
        for (int q = 1; q < EB_SLICES; ++q) s += sums[q][i];
        from_f32(dW[(long long)w * d + at], scale * s);
    }
}

// Up to EB_FEW tokens: one launch and no scratch. Against the three launches, 8192 words of 768 bf16: 64 tokens of a text 4.6 us for 17, 256 9.1 for 18,
// 512 14 for 18; all tokens one word, whose sum is one thread's per column: 11 for 16, 37 for 17, 71 for 18. An eager training pass, bound by the
// host at all of these, takes 51 us for 57. A CTA owns EB_FEW_WORDS words, its first warp finds their tokens and puts them in order of their words,
// then a thread adds up its columns token by token, in parts of EB_CHUNK tokens like the others.
constexpr int EB_FEW = 256, EB_FEW_WORDS = 32;
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_few_kernel(const long long *__restrict__ ids, const T *__restrict__ g, float scale, T *__restrict__ dW, int N, int V,
                                                        long long padding, int d) {
    __shared__ int tok[EB_FEW], word_of[EB_FEW], first[EB_FEW_WORDS + 1], next[EB_FEW_WORDS];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, v0 = blockIdx.x * EB_FEW_WORDS, words = min(EB_FEW_WORDS, V - v0);
    if (threadIdx.x < 32) {
        int word[EB_FEW / 32];
        next[lane] = 0;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < EB_FEW / 32; ++j) {
            const long long id = 32 * j + lane < N ? ids[32 * j + lane] : -1;
            const unsigned long long at = (unsigned long long)id - (unsigned)v0;
            word[j] = at < (unsigned)words && id != padding ? (int)at : -1;
        }
#pragma unroll
        for (int j = 0; j < EB_FEW / 32; ++j)
            if (word[j] >= 0) atomicAdd(&next[word[j]], 1);            // whole numbers: the order does not matter
        __syncwarp();
        const int count = next[lane];
        int inc = count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += up; }
        first[lane + 1] = inc;
        if (lane == 0) first[0] = 0;
        next[lane] = inc - count;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < EB_FEW / 32; ++j) {                        // the ones of a word ranked by the lanes before
            const bool here = word[j] >= 0;
            const unsigned who = __ballot_sync(0xffffffffu, here);
            if (who == 0u) continue;
            if (here) {
                const unsigned same = __match_any_sync(who, word[j]), before = same & ((1u << lane) - 1u);
                const int start = next[word[j]];
                tok[start + __popc(before)] = 32 * j + lane;
                word_of[start + __popc(before)] = word[j];
                __syncwarp(who);
                if (before == 0u) next[word[j]] = start + __popc(same);
            }
            __syncwarp();
        }
    }
    __syncthreads();
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    if (c >= d) return;
    for (int w = 0; w < words; ++w) {
        float none[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) none[q] = 0.f;
        if (first[w] == first[w + 1]) EbPack<T, VEC>::store(dW + (long long)(v0 + w) * d + c, none);
    }
    const int n = first[words];
    float acc[VEC], sum[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) { acc[q] = 0.f; sum[q] = 0.f; }
    constexpr int AHEAD = 16;
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
        typename EbPack<T, VEC>::Raw buf[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (i0 + j < n) buf[j] = EbPack<T, VEC>::load(g + (long long)tok[i0 + j] * d + c);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j;
            if (i >= n) break;
            float v[VEC];
            EbPack<T, VEC>::floats(buf[j], v);
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += v[q];
            const int w = word_of[i];
            const bool ends = i + 1 == first[w + 1];
            if (!ends && ((i - first[w] + 1) % EB_CHUNK) != 0) continue;
#pragma unroll
            for (int q = 0; q < VEC; ++q) { sum[q] += acc[q]; acc[q] = 0.f; }
            if (!ends) continue;
#pragma unroll
            for (int q = 0; q < VEC; ++q) sum[q] *= scale;
            EbPack<T, VEC>::store(dW + (long long)(v0 + w) * d + c, sum);
#pragma unroll
            for (int q = 0; q < VEC; ++q) sum[q] = 0.f;
        }
    }
}

// ------------------------------------------------------------------------------------------------ host
template <typename T, int VEC>
static int embed_fwd(const long long *ids, const void *W, float scale, void *y, long long N, int V, int d, cudaStream_t stream) {
    cudaError_t e = pdl_launch(embed_fwd_kernel<T, VEC>, dim3((unsigned)((N + 7) / 8)), dim3(256), 0, stream, ids, static_cast<const T *>(W), scale,
                               static_cast<T *>(y), N, V, d);
    if (e != cudaSuccess) { set_cuda_error(e, "embed_fwd launch"); return PGB_ERR_CUDA; }
    return check_launch("embed_fwd_kernel");
}
int embedding_fwd_launch(const long long *ids, const void *W, int dtype, float scale, void *y, long long N, int V, int d, cudaStream_t stream) {
    const bool wide = aligned(W, 16) && aligned(y, 16) && d % (dtype == PGB_F32 ? 4 : 8) == 0;
    if (dtype == PGB_F32) return wide ? embed_fwd<float, 4>(ids, W, scale, y, N, V, d, stream) : embed_fwd<float, 1>(ids, W, scale, y, N, V, d, stream);
    return wide ? embed_fwd<__nv_bfloat16, 8>(ids, W, scale, y, N, V, d, stream) : embed_fwd<__nv_bfloat16, 1>(ids, W, scale, y, N, V, d, stream);
}

static long long embed_chunks(long long N) { return (N + EB_CHUNK - 1) / EB_CHUNK; }
long long embedding_bwd_bytes(long long N, int V, int d) {
    if (N <= EB_FEW) return 0;
    auto up = [](long long x) { return (x + 255) / 256 * 256; };
    return up(8 * N) + up(8LL * (V + 1)) + up(embed_chunks(N) * 8 * d);
}
template <typename T, int VEC>
static int embed_few(const long long *ids, const void *g, float scale, void *dW, int N, int V, long long padding, int d, cudaStream_t stream) {
    const int cols = (d + VEC - 1) / VEC, nt = cols >= 256 ? 256 : (cols + 31) / 32 * 32;
    const cudaError_t e = pdl_launch(embed_few_kernel<T, VEC>, dim3((unsigned)((V + EB_FEW_WORDS - 1) / EB_FEW_WORDS), (unsigned)((cols + nt - 1) / nt)), dim3((unsigned)nt), 0,
                                     stream, ids, static_cast<const T *>(g), scale, static_cast<T *>(dW), N, V, padding, d);
    if (e != cudaSuccess) { set_cuda_error(e, "embed_few launch"); return PGB_ERR_CUDA; }
    return check_launch("embed_few_kernel");
}
template <typename T, int VEC>
static int embed_bwd(const void *g, float scale, void *dW, const int2 *order, const int2 *run, float *part, long long N, int V, int d,
                     cudaStream_t stream) {
    const int cols = (d + VEC - 1) / VEC, nt = cols >= 256 ? 256 : (cols + 31) / 32 * 32;
    const unsigned ny = (unsigned)((cols + nt - 1) / nt), chunks = (unsigned)embed_chunks(N);
    const int wide = EB_COLS * (VEC == 1 ? 1 : 4);                     // columns of a joining CTA
    cudaError_t e = pdl_launch(embed_sum_kernel<T, VEC>, dim3(chunks + (unsigned)((V + EB_ZERO - 1) / EB_ZERO), ny), dim3((unsigned)nt), 0, stream,
                               static_cast<const T *>(g), order, run, scale, static_cast<T *>(dW), part, (int)chunks, V, d);
    if (e == cudaSuccess && chunks > 1)
        e = pdl_launch(embed_join_kernel<T, VEC>, dim3(chunks - 1, (unsigned)((d + wide - 1) / wide)), dim3(EB_SLICES * EB_COLS), 0, stream, order, run,
                       static_cast<const float *>(part), scale, static_cast<T *>(dW), V, d);
    if (e != cudaSuccess) { set_cuda_error(e, "embed_sum launch"); return PGB_ERR_CUDA; }
    return check_launch("embed_sum_kernel");
}
int embedding_bwd_launch(const long long *ids, const void *g, int dtype, float scale, long long padding, void *dW, void *scratch, long long N, int V, int d,
                         cudaStream_t stream) {
    const bool wide = aligned(g, 16) && aligned(dW, 16) && d % (dtype == PGB_F32 ? 4 : 8) == 0;
    if (N <= EB_FEW) {
        if (dtype == PGB_F32)
            return wide ? embed_few<float, 4>(ids, g, scale, dW, (int)N, V, padding, d, stream) : embed_few<float, 1>(ids, g, scale, dW, (int)N, V, padding, d, stream);
        return wide ? embed_few<__nv_bfloat16, 8>(ids, g, scale, dW, (int)N, V, padding, d, stream)
                    : embed_few<__nv_bfloat16, 1>(ids, g, scale, dW, (int)N, V, padding, d, stream);
    }
    auto up = [](long long x) { return (x + 255) / 256 * 256; };
    char *s = static_cast<char *>(scratch);
    int2 *order = reinterpret_cast<int2 *>(s);
    int2 *run = reinterpret_cast<int2 *>(s + up(8 * N));
    float *part = reinterpret_cast<float *>(s + up(8 * N) + up(8LL * (V + 1)));
    int log_ctas = 7;                                                  // 128 CTAs, more where a CTA would own over EB_ROWS words
    while (((V - 1) >> log_ctas) + 1 > EB_ROWS) ++log_ctas;
    const int rows = (((V - 1) >> log_ctas) + 2) & ~1;                 // even: the list behind the histogram is 8-byte aligned
    const size_t smem = (size_t)EB_WARPS * rows * 4 + EB_WARPS * EB_LIST * 8;
    cudaError_t e = smem <= 49152 ? cudaSuccess
                  : cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EB_WARPS * EB_ROWS * 4 + EB_WARPS * EB_LIST * 8);
    if (e == cudaSuccess)
        e = pdl_launch(embed_sort_kernel, dim3(1u << log_ctas), dim3(EB_NT), smem, stream, ids, order, run, (int)N, V, padding, rows, log_ctas);
    if (e != cudaSuccess) { set_cuda_error(e, "embed_sort launch"); return PGB_ERR_CUDA; }
    if (dtype == PGB_F32)
        return wide ? embed_bwd<float, 4>(g, scale, dW, order, run, part, N, V, d, stream) : embed_bwd<float, 1>(g, scale, dW, order, run, part, N, V, d, stream);
    return wide ? embed_bwd<__nv_bfloat16, 8>(g, scale, dW, order, run, part, N, V, d, stream)
                : embed_bwd<__nv_bfloat16, 1>(g, scale, dW, order, run, part, N, V, d, stream);
}

}  // namespace pgb
