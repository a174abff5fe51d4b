// Attention of a step's new tokens over the paged cache, where each sequence brings a tree of drafted tokens (or one token, or a
// run of them): the general form, for every type and head size.
//
// Token t of a sequence with `pos0` earlier tokens sees keys 0 .. pos0 - 1 and, of the sequence's own new tokens (whose keys stand at
// places pos0, pos0 + 1, ... of the cache), number n where bit n % 64 of word n / 64 of its mask is set; without masks those up to
// itself.  out = sum_j p_j v_j, p = softmax over the keys it sees of scale q . k; a token that sees none gets zeros.  Keys and values are
// of the query's type or codes of 8 bits with a scale a row (page8.cuh).
// A block a (token, query head): four warps take every fourth key, each with a running maximum and sum of its own, and meet at the
// end.  A key that is not seen is not read.  Bound by the latency of its chain of keys: it is here for 32-bit queries and odd head sizes.
#include "../include/qwen3/cache_args.h"
#include "page8.cuh"

namespace {

constexpr int PAGE = Q3_PAGE_TOKENS, WARPS = 4, PER = 8;              // values of a head a lane: up to 256 in all

struct TreeArgs {
    const void *q, *k_pages, *v_pages;
    const uint8_t *k_scales, *v_scales;
    void* out;
    const int *seq_start, *seq_pos0, *page_table;
    const unsigned long long* tree;                // [tokens, words]; may be null
    int words, pages_per_seq, n_seqs, nq, nkv, d;
    int64_t n_pages;
    float scale;
};

template <typename T, bool F8>
__device__ __forceinline__ float value_at(const void* pages, int64_t cell, int d, int i) {
    if constexpr (F8) return __low2float(q3_half2_of(((const uint8_t*)pages)[cell * d + i]));
    else return to_f32<T>(((const T*)pages)[cell * d + i]);
}

template <typename T, bool F8>
__global__ void __launch_bounds__(WARPS * 32) tree_any_kernel(const TreeArgs a) {
    __shared__ float s_max[WARPS], s_sum[WARPS], s_out[WARPS][256];
    pdl_launch_dependents();
    pdl_wait();
    const int h = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d = a.d;
    const int64_t n = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (n >= a.seq_start[a.n_seqs]) return;
    int lo = 0, hi = a.n_seqs - 1;                 // the last sequence that starts at or before n
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.seq_start[mid] <= n) lo = mid; else hi = mid - 1;
    }
    const int seq = lo, first = a.seq_start[seq], n_new = a.seq_start[seq + 1] - first, pos0 = a.seq_pos0[seq];
    const int g = h / (a.nq / a.nkv), own = (int)(n - first);
    const unsigned long long* mask = a.tree != nullptr ? a.tree + n * a.words : nullptr;
    float q[PER], o[PER], m = -INFINITY, l = 0.0f;
    const T* row = (const T*)a.q + (n * a.nq + h) * d;
#pragma unroll
    for (int t = 0; t < PER; ++t) {
        q[t] = lane + 32 * t < d ? to_f32<T>(row[lane + 32 * t]) : 0.0f;
        o[t] = 0.0f;
    }
    const int keys = pos0 + (mask != nullptr ? min(n_new, a.words * 64) : own + 1);
    for (int j = warp; j < keys; j += WARPS) {
        const int x = j - pos0;
        if (x >= 0 && mask != nullptr && !(mask[x >> 6] >> (x & 63) & 1)) continue;
        if (j / PAGE >= a.pages_per_seq) break;
        const int64_t page = a.page_table[(int64_t)seq * a.pages_per_seq + j / PAGE];
        if (page < 0 || page >= a.n_pages) continue;
        const int64_t cell = (page * a.nkv + g) * PAGE + j % PAGE;
        float s = 0.0f;
#pragma unroll
        for (int t = 0; t < PER; ++t)
            if (lane + 32 * t < d) s += q[t] * value_at<T, F8>(a.k_pages, cell, d, lane + 32 * t);
        s = warp_sum(s) * a.scale;
        float vs = 1.0f;
        if constexpr (F8) {
            s *= q3_exp2i((int)a.k_scales[cell] - Q3_SCALE_BIAS);
            vs = q3_exp2i((int)a.v_scales[cell] - Q3_SCALE_BIAS);
        }
        const float m_new = fmaxf(m, s), old = m_new == m ? 1.0f : expf(m - m_new), p = s == -INFINITY ? 0.0f : expf(s - m_new);
        m = m_new;
        l = l * old + p;
#pragma unroll
        for (int t = 0; t < PER; ++t)
            if (lane + 32 * t < d) o[t] = o[t] * old + p * (vs * value_at<T, F8>(a.v_pages, cell, d, lane + 32 * t));
    }
#pragma unroll
    for (int t = 0; t < PER; ++t)
        if (lane + 32 * t < d) s_out[warp][lane + 32 * t] = o[t];
    if (lane == 0) {
        s_max[warp] = m;
        s_sum[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.0f, w[WARPS];
    for (int i = 0; i < WARPS; ++i) top = fmaxf(top, s_max[i]);
    for (int i = 0; i < WARPS; ++i) {
        w[i] = s_max[i] == top ? 1.0f : expf(s_max[i] - top);         // (no key seen by any warp: sums of zero)
        sum += s_sum[i] * w[i];
    }
    T* to = (T*)a.out + (n * a.nq + h) * d;
    for (int i = threadIdx.x; i < d; i += WARPS * 32) {
        float v = 0.0f;
        for (int k = 0; k < WARPS; ++k) v += s_out[k][i] * w[k];
        to[i] = from_f32<T>(sum == 0.0f ? 0.0f : v / sum);
    }
}

template <typename T, bool F8>
int launch(const TreeArgs& a, int64_t n_tokens, cudaStream_t stream) {
    const dim3 grid(a.nq, (unsigned)(n_tokens < 65535 ? n_tokens : 65535), (unsigned)((n_tokens + 65534) / 65535));
    return (int)q3_launch(tree_any_kernel<T, F8>, grid, dim3(WARPS * 32), 0, stream, a);
}

int attend(const q3_attention_tree_args& x, bool f32) {
    const TreeArgs a = {x.q, x.k_pages, x.v_pages, (const uint8_t*)x.k_scales, (const uint8_t*)x.v_scales, x.out, (const int*)x.seq_start,
                        (const int*)x.seq_pos0, (const int*)x.page_table, (const unsigned long long*)x.tree, x.words, x.pages_per_seq, x.n_seqs, x.nq, x.nkv,
                        x.d, x.n_pages, (float)x.scale};
    if (a.n_seqs <= 0 || x.n_tokens <= 0) return 0;
    if (a.nq <= 0 || a.nkv <= 0 || a.nq % a.nkv != 0 || a.d <= 0 || a.d > 256 || (a.tree != nullptr && a.words <= 0)) return Q3_ERR_BAD_SIZE;
    if (x.n_tokens > (int64_t)65535 * 65535) return Q3_ERR_TOO_LARGE;
    const bool f8 = a.k_scales != nullptr;
    cudaStream_t s = (cudaStream_t)x.stream;
    if (f32) return f8 ? launch<float, true>(a, x.n_tokens, s) : launch<float, false>(a, x.n_tokens, s);
    return f8 ? launch<bf16, true>(a, x.n_tokens, s) : launch<bf16, false>(a, x.n_tokens, s);
}

}  // namespace

Q3_EXPORT int q3_attention_tree_any_f32(const q3_attention_tree_args* a) { return attend(*a, true); }
Q3_EXPORT int q3_attention_tree_any_bf16(const q3_attention_tree_args* a) { return attend(*a, false); }
