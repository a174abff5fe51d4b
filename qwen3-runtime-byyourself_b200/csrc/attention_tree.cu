// Attention of a step's new tokens over the paged cache, where each sequence brings a tree of drafted tokens (or one token, or a
// run of them): the general form, for every type and head size.
//
// Token t of a sequence with `pos0` earlier tokens sees keys 0 .. pos0 - 1 and, of the sequence's own new tokens (whose keys stand at
// places pos0, pos0 + 1, ... of the cache), number n where bit n % 64 of word n / 64 of its mask is set; without masks those up to
// itself.  out = sum_j p_j v_j, p = softmax over the keys it sees of scale q . k; a token that sees none gets zeros.  Keys and values are
// of the query's type or codes of 8 bits with a scale a row (page8.cuh).
// A block a (token, query head): each of its warps takes every eighth stretch of 32 keys, with a running maximum and sum of its own, and they meet at the
// end.  The stretch's scores are made eight keys at a time, so that many loads are on their way; then its maximum and its weights, a key a lane; then
// its values are added up, eight at a time again.  A key that is not seen is not read.  It is here for 32-bit queries and odd head sizes.  Its grid
// bounds it: one token of 32 heads is 32 blocks on 148 SMs, each with a chain of loads over all keys, and rows that share a head's keys read them from the L2 again.
// One token of 32 heads over 8 and 2,000 keys, 32-bit, 102 us (one key after the other 443; the floor is 2.5), 8 sequences of up to 2,000 and 8 tokens each 322
// (floor 9.3); bfloat16 heads of 96 over 8 bits, 8 sequences of up to 4,000 and one token each 340 (floor 5.1), heads of 256 517 (7.7).
#include "../include/qwen3/cache_args.h"
#include "page8.cuh"

namespace {

constexpr int PAGE = Q3_PAGE_TOKENS, WARPS = 8, KEYS = 8;                     // keys whose loads are on their way together

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

// Value i of a row, zero beyond its end (without a branch: loads of several rows go out together).
template <typename T, bool F8>
__device__ __forceinline__ float value_at(const void* pages, int64_t cell, int d, int i) {
    const int64_t at = cell * d + min(i, d - 1);
    float v;
    if constexpr (F8) v = __low2float(q3_half2_of(((const uint8_t*)pages)[at]));
    else v = to_f32<T>(((const T*)pages)[at]);
    return i < d ? v : 0.0f;
}

// PER: values of a head a lane.
template <typename T, bool F8, int PER>
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
    for (int j0 = warp * 32; j0 < keys && j0 / PAGE < a.pages_per_seq; j0 += WARPS * 32) {
        const int64_t page = a.page_table[(int64_t)seq * a.pages_per_seq + j0 / PAGE];
        if (page < 0 || page >= a.n_pages) continue;
        const int64_t cell0 = (page * a.nkv + g) * PAGE + j0 % PAGE;
        const int x = j0 + lane - pos0;
        const bool sees = j0 + lane < keys && (x < 0 || mask == nullptr || (mask[x >> 6] >> (x & 63) & 1));
        const unsigned seen = __ballot_sync(0xffffffffu, sees);
        if (seen == 0) continue;
        const int some = __ffs(seen) - 1;          // stands in for keys that are not seen
        float factor = a.scale, vs = 1.0f, s = -INFINITY;
        if (F8 && sees) {
            factor = q3_exp2i((int)a.k_scales[cell0 + lane] - Q3_SCALE_BIAS);
            vs = q3_exp2i((int)a.v_scales[cell0 + lane] - Q3_SCALE_BIAS);
        }
#pragma unroll 1
        for (int k0 = 0; k0 < 32; k0 += KEYS) {
            if ((seen >> k0 & ((1u << KEYS) - 1u)) == 0) continue;
            float dot[KEYS];
#pragma unroll
            for (int k = 0; k < KEYS; ++k) {
                const int64_t cell = cell0 + (seen >> (k0 + k) & 1u ? k0 + k : some);
                dot[k] = 0.0f;
#pragma unroll
                for (int t = 0; t < PER; ++t) dot[k] += q[t] * value_at<T, F8>(a.k_pages, cell, d, lane + 32 * t);
            }
#pragma unroll
            for (int k = 0; k < KEYS; ++k) {
                const float sum = warp_sum(dot[k]);
                if (lane == k0 + k) s = sum;
            }
        }
        if (F8) s *= a.scale;
        s = sees ? s * factor : -INFINITY;
        const float m_new = fmaxf(m, warp_max(s)), old = m_new == m ? 1.0f : expf(m - m_new), p = s == -INFINITY ? 0.0f : expf(s - m_new);
        m = m_new;
        l = l * old + warp_sum(p);
        const float pv = p * vs;
#pragma unroll
        for (int t = 0; t < PER; ++t) o[t] *= old;
#pragma unroll 1
        for (int k0 = 0; k0 < 32; k0 += KEYS) {
            if ((seen >> k0 & ((1u << KEYS) - 1u)) == 0) continue;
#pragma unroll
            for (int k = 0; k < KEYS; ++k) {
                const bool here = seen >> (k0 + k) & 1u;
                const int64_t cell = cell0 + (here ? k0 + k : some);
                const float w = __shfl_sync(0xffffffffu, pv, k0 + k);
#pragma unroll
                for (int t = 0; t < PER; ++t) {
                    const float v = value_at<T, F8>(a.v_pages, cell, d, lane + 32 * t);
                    o[t] = here ? fmaf(w, v, o[t]) : o[t];
                }
            }
        }
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
    const dim3 block(WARPS * 32);
    return (int)(a.d <= 64    ? q3_launch(tree_any_kernel<T, F8, 2>, grid, block, 0, stream, a)
                 : a.d <= 128 ? q3_launch(tree_any_kernel<T, F8, 4>, grid, block, 0, stream, a)
                              : q3_launch(tree_any_kernel<T, F8, 8>, grid, block, 0, stream, a));
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
