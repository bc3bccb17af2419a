// What stands between a model's logits and the draw: penalties for words seen before, biases of single words, and a mask of the words a grammar allows.
// For word v of row b, with n the times v stands among the generated ids and m those and the prompt's together,
//
//     s = l;   m > 0: s = s > 0 ? s / r : s r;   n > 0: s = s - f n - p;   s += biases of v, in their order;   not allowed: s = -inf
//
// in fp32, each operation rounded. Ids outside 0 .. V-1 (padding) count nowhere.
//
// A CTA owns a slice of a row's words: it counts the row's ids that fall into the slice in shared memory (a row's history is read once a slice, from the L2 but
// for the first time), while the slice's logits are on their way. No table of counts in memory, nothing carried from one call to the next. Counts are whole
// numbers, so the order of the atomics changes nothing; a word's biases are added up by the first entry that names it.
#include "common.cuh"

namespace pgb {

constexpr int ADJ_MOST_BIAS = 1024;

__device__ __forceinline__ int list_length(const TokenList &t, long long b) {
    if (t.n == 0 || t.lengths == nullptr) return t.n;
    const long long n = t.lengths[b * t.length_stride];
    return n < 0 ? 0 : n > t.n ? t.n : (int)n;
}

// NT threads, VPT words each: slices of NT VPT words. SEEN: 0x80000000 marks a word of the prompt, the rest counts the generated ones.
template <typename T_, int NT, int VPT>
__global__ void __launch_bounds__(NT) adjust_logits_kernel(AdjustLogits a, int slices) {
    constexpr int S = NT * VPT;
    constexpr uint32_t IN_PROMPT = 0x80000000u;
    extern __shared__ uint32_t adj_smem[];
    uint32_t *count = adj_smem;                                       // [S]
    float *sbias = reinterpret_cast<float *>(adj_smem + S);           // [S] with biases
    int *bid = reinterpret_cast<int *>(adj_smem + 2 * S);             // [nb]: place in the slice, -1 outside
    float *bval = reinterpret_cast<float *>(bid + a.nb);
    const int tid = threadIdx.x;
    const long long b = blockIdx.x / slices;
    const int v0 = (int)(blockIdx.x % slices) * S;
    pdl_launch_dependents();
    pdl_wait();

    const T_ *row = reinterpret_cast<const T_ *>(a.logits) + b * a.stride;
    float l[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int v = v0 + tid + i * NT;
        l[i] = v < a.V ? to_f32(row[v]) : 0.f;
    }
    const int np = list_length(a.prompt, b), ng = list_length(a.made, b);
#pragma unroll
    for (int i = 0; i < VPT; ++i) count[tid + i * NT] = 0u;
    if (a.nb > 0) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) sbias[tid + i * NT] = 0.f;
        for (int j = tid; j < a.nb; j += NT) {
            const long long at = a.bias_ids[b * a.bias_stride + j] - v0;
            const bool in = at >= 0 && at < S && at + v0 < a.V;
            bid[j] = in ? (int)at : -1;
            bval[j] = a.bias[b * a.bias_stride + j];
        }
    }
    __syncthreads();
    const long long *ids = a.prompt.ids + b * a.prompt.stride;
#pragma unroll 8
    for (int j = tid; j < np; j += NT) {
        const long long at = ids[j] - v0;
        if (at >= 0 && at < S && !(count[at] & IN_PROMPT)) atomicOr(&count[at], IN_PROMPT);
    }
    ids = a.made.ids + b * a.made.stride;
#pragma unroll 8
    for (int j = tid; j < ng; j += NT) {
        const long long at = ids[j] - v0;
        if (at >= 0 && at < S) atomicAdd(&count[at], 1u);
    }
    for (int j = tid; j < a.nb; j += NT) {
        const int at = bid[j];
        if (at < 0) continue;
        bool first = true;
        for (int i = 0; i < j; ++i) first = first && bid[i] != at;
        if (!first) continue;
        float s = bval[j];
        for (int i = j + 1; i < a.nb; ++i)
            if (bid[i] == at) s += bval[i];
        sbias[at] = s;
    }
    __syncthreads();

    const float r = a.repetition.at ? a.repetition.at[b] : a.repetition.all, f = a.frequency.at ? a.frequency.at[b] : a.frequency.all,
                p = a.presence.at ? a.presence.at[b] : a.presence.all;
    float *out = a.out + b * (long long)a.V;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int at = tid + i * NT, v = v0 + at;
        if (v >= a.V) break;
        float s = l[i];
        const uint32_t c = count[at];
        if (c != 0u) {
            s = s > 0.f ? __fdiv_rn(s, r) : __fmul_rn(s, r);
            const uint32_t n = c & ~IN_PROMPT;
            if (n != 0u) s = __fsub_rn(__fsub_rn(s, __fmul_rn(f, (float)n)), p);
        }
        if (a.nb > 0) s = __fadd_rn(s, sbias[at]);
        bool ok = true;
        if (a.mask_kind == 1) ok = (reinterpret_cast<const uint32_t *>(a.mask)[b * a.mask_stride + (v >> 5)] >> (v & 31)) & 1u;
        else if (a.mask_kind == 2) ok = reinterpret_cast<const unsigned char *>(a.mask)[b * a.mask_stride + v] != 0;
        out[v] = ok ? s : -INFINITY;
    }
}

template <typename T_, int NT, int VPT>
static cudaError_t adjust_go(const AdjustLogits &a, cudaStream_t stream) {
    constexpr int S = NT * VPT;
    const int slices = (a.V + S - 1) / S;
    const size_t smem = (size_t)S * 4 * (a.nb > 0 ? 2 : 1) + (size_t)a.nb * 8;
    return pdl_launch(adjust_logits_kernel<T_, NT, VPT>, dim3((unsigned)(a.B * slices)), dim3(NT), smem, stream, a, slices);
}
int adjust_logits_launch(const AdjustLogits &a, cudaStream_t stream) {
    const bool many = a.prompt.n + a.made.n > 4096;
    cudaError_t e;
    if (a.dtype == PGB_BF16) e = many ? adjust_go<__nv_bfloat16, 1024, 4>(a, stream) : adjust_go<__nv_bfloat16, 256, 8>(a, stream);
    else e = many ? adjust_go<float, 1024, 4>(a, stream) : adjust_go<float, 256, 8>(a, stream);
    if (e != cudaSuccess) { set_cuda_error(e, "adjust_logits launch"); return PGB_ERR_CUDA; }
    return check_launch("adjust_logits_kernel");
}

}  // namespace pgb
