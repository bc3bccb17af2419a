// Embedding lookup with scaling, y_n = scale w_{id_n}, and its gradient dw_v = scale sum_{n: id_n = v} g_n by sorted tokens: no atomics on
// the sums, so the same call gives the same bits, and a word's gradients are added in fp32 and rounded once.
//   Both directions move bytes and compute nothing to speak of: the lookup reads and writes N rows, the gradient reads N rows and writes V.
//   The gradient is three launches, each a programmatic dependent of the one before:
//   embed_sort_kernel  a CTA owns a range of the vocabulary and reads all ids once (8 N bytes from the L2), which tells it its own tokens
//                      in order and how many tokens belong to lower words: a stable counting sort without a word exchanged between CTAs.
//   embed_sum_kernel   the sorted tokens in chunks of EB_CHUNK, whatever words they hold, so a frequent word is spread over many CTAs: a run
//                      that lies in one chunk is finished there, one that crosses a border leaves fp32 partial sums. Further CTAs write the
//                      zeros of words that no token has.
//   embed_join_kernel  adds the partial sums of the runs that cross borders, in order.
#include "common.cuh"

namespace pgb {

constexpr int EB_WARPS = 32, EB_NT = EB_WARPS * 32, EB_ROWS = 512, EB_LIST = 64;   // sort: warps, most words a CTA owns, a warp's list of its tokens
constexpr int EB_CHUNK = 32, EB_ZERO = 32;                            // sorted tokens of a summing CTA, words of a zeroing one

// 16 bytes of T, or one element where a row is no whole number of them
template <typename T, int VEC> struct EbPack { static __device__ __forceinline__ void load(const T *p, float (&v)[VEC]);
                                               static __device__ __forceinline__ void store(T *p, const float (&v)[VEC]); };
template <typename T> struct EbPack<T, 1> {
    static __device__ __forceinline__ void load(const T *p, float (&v)[1]) { v[0] = to_f32(*p); }
    static __device__ __forceinline__ void store(T *p, const float (&v)[1]) { from_f32(*p, v[0]); }
};
template <> struct EbPack<float, 4> {
    static __device__ __forceinline__ void load(const float *p, float (&v)[4]) { *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(p); }
    static __device__ __forceinline__ void store(float *p, const float (&v)[4]) { *reinterpret_cast<float4 *>(p) = *reinterpret_cast<const float4 *>(v); }
};
template <> struct EbPack<__nv_bfloat16, 8> {
    static __device__ __forceinline__ void load(const __nv_bfloat16 *p, float (&v)[8]) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(p);
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&raw);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __bfloat1622float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
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
        EbPack<T, VEC>::load(w + c, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = in ? scale * v[i] : __int_as_float(0x7fffffff);
        EbPack<T, VEC>::store(out + c, v);
    }
}

// ------------------------------------------------------------------------------------------------ gradient: the tokens in order of their words
// order [N]: token numbers, by word, ascending within a word; first [V + 1]: where a word's begin. Tokens whose id is outside the table
// or the padding word are left out.
__global__ void __launch_bounds__(EB_NT, 1) embed_sort_kernel(const long long *__restrict__ ids, int *__restrict__ order, int *__restrict__ first, int N, int V,
                                                              long long padding, int rows_per) {
    extern __shared__ int eb_smem[];
    int *hist = eb_smem;                                               // [warps][rows_per]: a warp's tokens of a word, then where its next one goes
    int2 *list = reinterpret_cast<int2 *>(hist + EB_WARPS * rows_per);
    __shared__ int below[EB_WARPS], scan[EB_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lo = blockIdx.x * rows_per, rows = min(rows_per, V - lo);
    for (int i = threadIdx.x; i < EB_WARPS * rows_per; i += EB_NT) hist[i] = 0;
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    // a warp reads a contiguous share of the ids, 32 at a time, four loads in flight
    const int share = ((N + EB_WARPS - 1) / EB_WARPS + 31) & ~31, from = min(N, warp * share), to = min(N, from + share);
    const unsigned lt = (1u << lane) - 1u;
    int2 *mine = list + warp * EB_LIST;
    int n_below = 0, n_found = 0;
    auto visit = [&](auto &&take) {
        for (int n0 = from; n0 < to; n0 += 128) {
            long long id[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { const int n = n0 + 32 * j + lane; id[j] = n < to ? ids[n] : -1; }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool use = id[j] >= 0 && id[j] < V && id[j] != padding;
                const bool here = use && id[j] >= lo && id[j] < lo + rows;
                take(n0 + 32 * j + lane, (int)id[j] - lo, here, use && id[j] < lo);
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
        for (int w = 0; w < EB_WARPS; ++w) total += hist[w * rows_per + r0];
    int inc = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += up; }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    int base = 0;
    for (int w = 0; w < EB_WARPS; ++w) { base += below[w]; if (w < warp) base += scan[w]; }
    int at = base + inc - total;
    if (r0 < rows) {
        first[lo + r0] = at;
        if (lo + r0 == V - 1) first[V] = at + total;
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
            order[start + __popc(same & lt)] = n;
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
template <typename T, int VEC>
__global__ void embed_sum_kernel(const long long *__restrict__ ids, const T *__restrict__ g, const int *__restrict__ order, const int *__restrict__ first,
                                 float scale, T *__restrict__ dW, float *__restrict__ part, int chunks, int V, int d) {
    __shared__ int tok[EB_CHUNK], word[EB_CHUNK];
    pdl_wait();
    pdl_launch_dependents();
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
    float v[VEC];
    if ((int)blockIdx.x >= chunks) {                                   // words without a token
        const int v0 = (blockIdx.x - chunks) * EB_ZERO;
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 0.f;
        if (c < d)
            for (int w = v0; w < v0 + EB_ZERO && w < V; ++w)
                if (first[w] == first[w + 1]) EbPack<T, VEC>::store(dW + (long long)w * d + c, v);
        return;
    }
    const int a = blockIdx.x * EB_CHUNK, b = min(a + EB_CHUNK, first[V]);
    if (a >= b) return;
    for (int i = threadIdx.x; i < b - a; i += blockDim.x) {
        const int n = order[a + i];
        tok[i] = n;
        word[i] = (int)ids[n];
    }
    __syncthreads();
    if (c >= d) return;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    const int n = b - a;
    constexpr int AHEAD = 8;
    float buf[AHEAD][VEC];
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (i0 + j < n) EbPack<T, VEC>::load(g + (long long)tok[i0 + j] * d + c, buf[j]);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j;
            if (i >= n) break;
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] += buf[j][q];
            const int w = word[i];
            if (i + 1 < n && word[i + 1] == w) continue;               // the run goes on
            const int from = first[w], to = first[w + 1];
            if (from >= a && to <= b) {
#pragma unroll
                for (int q = 0; q < VEC; ++q) acc[q] *= scale;
                EbPack<T, VEC>::store(dW + (long long)w * d + c, acc);
            } else {
                float *p = part + ((long long)blockIdx.x * 2 + (from >= a)) * d + c;
#pragma unroll
                for (int q = 0; q < VEC; ++q) p[q] = acc[q];
            }
#pragma unroll
            for (int q = 0; q < VEC; ++q) acc[q] = 0.f;
        }
    }
}
// the run that begins in this chunk and goes on behind it: its partial sums, in order
template <typename T, int VEC>
__global__ void embed_join_kernel(const long long *__restrict__ ids, const int *__restrict__ order, const int *__restrict__ first,
                                  const float *__restrict__ part, float scale, T *__restrict__ dW, int V, int d) {
    pdl_wait();
    pdl_launch_dependents();
    const int end = (blockIdx.x + 1) * EB_CHUNK;
    if (end >= first[V]) return;
    const int w = (int)ids[order[end]], from = first[w], to = first[w + 1];
    if (from >= end || from < end - EB_CHUNK) return;                  // no run crosses this border, or it began further ahead
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC, last = (to - 1) / EB_CHUNK;
    if (c >= d) return;
    float acc[VEC];
    const float *p = part + ((long long)blockIdx.x * 2 + 1) * d + c;
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] = p[q];
#pragma unroll 8
    for (int j = blockIdx.x + 1; j <= last; ++j) {
        const float *o = part + (long long)j * 2 * d + c;
#pragma unroll
        for (int q = 0; q < VEC; ++q) acc[q] += o[q];
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) acc[q] *= scale;
    EbPack<T, VEC>::store(dW + (long long)w * d + c, acc);
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
    auto up = [](long long x) { return (x + 255) / 256 * 256; };
    return up(4 * N) + up(4LL * (V + 1)) + up(embed_chunks(N) * 8 * d);
}
template <typename T, int VEC>
static int embed_bwd(const long long *ids, const void *g, float scale, void *dW, const int *order, const int *first, float *part, long long N, int V, int d,
                     cudaStream_t stream) {
    const int cols = (d + VEC - 1) / VEC, nt = cols >= 256 ? 256 : (cols + 31) / 32 * 32;
    const unsigned ny = (unsigned)((cols + nt - 1) / nt), chunks = (unsigned)embed_chunks(N);
    cudaError_t e = pdl_launch(embed_sum_kernel<T, VEC>, dim3(chunks + (unsigned)((V + EB_ZERO - 1) / EB_ZERO), ny), dim3((unsigned)nt), 0, stream, ids,
                               static_cast<const T *>(g), order, first, scale, static_cast<T *>(dW), part, (int)chunks, V, d);
    if (e == cudaSuccess && chunks > 1)
        e = pdl_launch(embed_join_kernel<T, VEC>, dim3(chunks - 1, ny), dim3((unsigned)nt), 0, stream, ids, order, first, part, scale, static_cast<T *>(dW), V, d);
    if (e != cudaSuccess) { set_cuda_error(e, "embed_sum launch"); return PGB_ERR_CUDA; }
    return check_launch("embed_sum_kernel");
}
int embedding_bwd_launch(const long long *ids, const void *g, int dtype, float scale, long long padding, void *dW, void *scratch, long long N, int V, int d,
                         cudaStream_t stream) {
    auto up = [](long long x) { return (x + 255) / 256 * 256; };
    char *s = static_cast<char *>(scratch);
    int *order = reinterpret_cast<int *>(s), *first = reinterpret_cast<int *>(s + up(4 * N));
    float *part = reinterpret_cast<float *>(s + up(4 * N) + up(4LL * (V + 1)));
    const int sms = sm_count();
    int rows = (V + sms - 1) / sms;
    if (rows > EB_ROWS) rows = EB_ROWS;
    rows = (rows + 1) & ~1;                                            // the list behind the histogram is 8-byte aligned
    const size_t smem = (size_t)EB_WARPS * rows * 4 + EB_WARPS * EB_LIST * 8;
    cudaError_t e = cudaFuncSetAttribute(embed_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EB_WARPS * EB_ROWS * 4 + EB_WARPS * EB_LIST * 8);
    if (e == cudaSuccess)
        e = pdl_launch(embed_sort_kernel, dim3((unsigned)((V + rows - 1) / rows)), dim3(EB_NT), smem, stream, ids, order, first, (int)N, V, padding, rows);
    if (e != cudaSuccess) { set_cuda_error(e, "embed_sort launch"); return PGB_ERR_CUDA; }
    const bool wide = aligned(g, 16) && aligned(dW, 16) && d % (dtype == PGB_F32 ? 4 : 8) == 0;
    if (dtype == PGB_F32)
        return wide ? embed_bwd<float, 4>(ids, g, scale, dW, order, first, part, N, V, d, stream) : embed_bwd<float, 1>(ids, g, scale, dW, order, first, part, N, V, d, stream);
    return wide ? embed_bwd<__nv_bfloat16, 8>(ids, g, scale, dW, order, first, part, N, V, d, stream)
                : embed_bwd<__nv_bfloat16, 1>(ids, g, scale, dW, order, first, part, N, V, d, stream);
}

}  // namespace pgb
