// Rows of the paged cache: written from a projection (normed, rotated, and quantised to 8 bits where the cache is kept so),
// read back, and moved after a step with drafted tokens.
//
// All three move bytes and compute next to nothing, so each is bound by memory; what each row costs:
//   append   reads (nq + 2 nkv) d values of the projection and d / 2 angles a token, writes nq d values and 2 nkv rows;
//   read     reads d + 1 bytes a row and writes 2 d (bfloat16);
//   keep     reads and writes the rows that move.
// Norm and rotation as in attention.cu's qkv_prepare (src/model/self_attention.cpp:122-152): y = x / sqrt(mean(x^2) + eps) w
// over a head, values i and i + r/2 of the first r turned by the angle of the token's position.  A token's place in the
// cache is given beside its position: drafted tokens of a tree stand side by side at places of their own, several at one position.
#include "page8.cuh"

namespace {

constexpr int PAGE = Q3_PAGE_TOKENS;

// Where the rows of token n go: the page and the place in it; false: nowhere (no such page).
__device__ __forceinline__ bool place_of(const int* __restrict__ table, int pages_per_seq, int64_t n_pages, int seq, int place, int64_t& page, int& at) {
    const int i = place / PAGE;
    if (place < 0 || i >= pages_per_seq) return false;
    page = table[(int64_t)seq * pages_per_seq + i];
    at = place % PAGE;
    return page >= 0 && page < n_pages;
}

struct AppendArgs {
    const void* qkv;
    void *q_out, *k_pages, *v_pages;
    uint8_t *k_scales, *v_scales;                  // a cache in 8 bits
    const float *q_norm, *k_norm, *cos_tab, *sin_tab;
    const int *token_seq, *token_pos, *token_place, *page_table;
    int pages_per_seq, nq, nkv, d, rot, norm_once;
    int64_t n_pages, n_tokens, row;                // row: values of a row of qkv
    float eps;
};

// ---- any head size up to 256: a warp a head, a value a lane and turn
template <typename T, bool F8>
__global__ void __launch_bounds__(256) append_any_kernel(const AppendArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int heads = a.nq + 2 * a.nkv, lane = threadIdx.x & 31;
    const int64_t vec = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (vec >= a.n_tokens * heads) return;
    const int64_t n = vec / heads;
    const int h = (int)(vec - n * heads), d = a.d;
    const bool is_q = h < a.nq, is_v = h >= a.nq + a.nkv;
    const T* x = (const T*)a.qkv + n * a.row + (int64_t)h * d;
    const float* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
    const int half = a.rot >> 1, pos = a.token_pos[n];
    constexpr int PER = 8;                                          // 256 / 32
    float sq = 0.0f, y[PER];
#pragma unroll
    for (int t = 0; t < PER; ++t) {
        const int i = lane + 32 * t;
        y[t] = i < d ? to_f32<T>(x[i]) : 0.0f;
        sq += y[t] * y[t];
    }
    const float inv = w != nullptr ? rsqrtf(warp_sum(sq) / (float)d + a.eps) : 1.0f;
    auto normed = [&](int i, float v) {
        if (w == nullptr) return v;
        return a.norm_once ? v * inv * w[i] : round_to<T>(round_to<T>(v * inv) * w[i]);
    };
    float top = 0.0f;
#pragma unroll
    for (int t = 0; t < PER; ++t) {
        const int i = lane + 32 * t;
        if (i >= d) break;
        float v = normed(i, y[t]);
        if (!is_v && a.cos_tab != nullptr && i < a.rot) {
            const int j = i < half ? i : i - half, other = i < half ? i + half : j;
            const float u = normed(other, to_f32<T>(x[other])), c = a.cos_tab[(int64_t)pos * half + j], s = a.sin_tab[(int64_t)pos * half + j];
            v = i < half ? v * c - u * s : v * c + u * s;
        }
        y[t] = F8 && !a.norm_once ? round_to<T>(v) : v;
        if (q3_is_number(y[t])) top = fmaxf(top, fabsf(y[t]));
    }
    if (is_q) {
        T* to = (T*)a.q_out + (n * a.nq + h) * d;
#pragma unroll
        for (int t = 0; t < PER; ++t)
            if (lane + 32 * t < d) to[lane + 32 * t] = from_f32<T>(y[t]);
        return;
    }
    int64_t page;
    int at;
    if (!place_of(a.page_table, a.pages_per_seq, a.n_pages, a.token_seq[n], a.token_place[n], page, at)) return;
    const int g = is_v ? h - a.nq - a.nkv : h - a.nq;
    const int64_t cell = (page * a.nkv + g) * PAGE + at;
    if constexpr (F8) {
        const int k = q3_scale_exponent(warp_max(top));
        uint8_t* to = (uint8_t*)(is_v ? a.v_pages : a.k_pages) + cell * d;
#pragma unroll
        for (int t = 0; t < PER; ++t)
            if (lane + 32 * t < d) to[lane + 32 * t] = (uint8_t)q3_codes2(y[t], 0.0f, q3_exp2i(-k));
        if (lane == 0) (is_v ? a.v_scales : a.k_scales)[cell] = (uint8_t)(k + Q3_SCALE_BIAS);
    } else {
        T* to = (T*)(is_v ? a.v_pages : a.k_pages) + cell * d;
#pragma unroll
        for (int t = 0; t < PER; ++t)
            if (lane + 32 * t < d) to[lane + 32 * t] = from_f32<T>(y[t]);
    }
}

template <typename T, bool F8>
int launch_append(const AppendArgs& a, cudaStream_t stream) {
    const int64_t vecs = a.n_tokens * (a.nq + 2 * a.nkv);
    const int64_t blocks = (vecs + 7) / 8;
    if (blocks > 0x7fffffff) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch(append_any_kernel<T, F8>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

// ---- the cached rows of sequences as pages of T, page j of sequence s at s * out_pages + j
template <typename T>
__global__ void __launch_bounds__(256)
read_kernel(const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const uint8_t* __restrict__ k_scales,
            const uint8_t* __restrict__ v_scales, const int* __restrict__ page_table, int pages_per_seq, const int* __restrict__ seq_end,
            int64_t n_pages, T* __restrict__ k_out, T* __restrict__ v_out, int out_pages, int nkv, int d) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.z, j = blockIdx.x, g = blockIdx.y, live = min(PAGE, seq_end[seq] - j * PAGE);
    if (live <= 0 || j >= pages_per_seq) return;
    const int64_t page = page_table[(int64_t)seq * pages_per_seq + j];
    if (page < 0 || page >= n_pages) return;
    const int64_t from = (page * nkv + g) * PAGE, to = (((int64_t)seq * out_pages + j) * nkv + g) * PAGE;
    for (int i = threadIdx.x; i < PAGE * d; i += blockDim.x) {
        const int r = i / d;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const uint8_t code = (side ? v_pages : k_pages)[from * d + i], scale = (side ? v_scales : k_scales)[from + r];
            const float v = __low2float(q3_half2_of(code)) * q3_exp2i((int)scale - Q3_SCALE_BIAS);
            (side ? v_out : k_out)[to * d + i] = from_f32<T>(r < live ? v : 0.0f);
        }
    }
}

// ---- rows pos0 + path[i] to pos0 + i, in every area (a layer's keys or values)
// A thread owns the same 16 bytes of every row of a kv head (the scales: a byte) and walks the path, which ascends: the row that
// it writes has been read by then, if it is one of the path's.
__global__ void __launch_bounds__(256)
keep_kernel(unsigned char* __restrict__ store, uint8_t* __restrict__ scales, int64_t n_pages, int nkv, int row_bytes,
            const int* __restrict__ page_table, int pages_per_seq, const int* __restrict__ seq_pos0, const int* __restrict__ path, int path_len) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.y, packets = row_bytes / 16, per_head = packets + (scales != nullptr ? 1 : 0);
    const int64_t area = blockIdx.x;
    const int pos0 = seq_pos0[seq];
    for (int i = threadIdx.x; i < nkv * per_head; i += blockDim.x) {
        const int g = i / per_head, c = i % per_head;
        for (int n = 0; n < path_len; ++n) {
            const int node = path[(int64_t)seq * path_len + n];
            if (node < 0) break;
            int64_t from_page, to_page;
            int from_at, to_at;
            if (node <= n || !place_of(page_table, pages_per_seq, n_pages, seq, pos0 + node, from_page, from_at) ||
                !place_of(page_table, pages_per_seq, n_pages, seq, pos0 + n, to_page, to_at))
                continue;
            const int64_t from = ((area * n_pages + from_page) * nkv + g) * PAGE + from_at, to = ((area * n_pages + to_page) * nkv + g) * PAGE + to_at;
            if (c == packets) scales[to] = scales[from];
            else *reinterpret_cast<uint4*>(store + to * row_bytes + c * 16) = *reinterpret_cast<const uint4*>(store + from * row_bytes + c * 16);
        }
    }
}

int append(AppendArgs a, bool f32, bool f8, void* stream) {
    if (a.n_tokens <= 0) return 0;
    if (a.nq <= 0 || a.nkv <= 0 || a.d <= 0 || a.d > 256 || a.rot < 0 || a.rot > a.d || (a.rot & 1) || a.row < (int64_t)(a.nq + 2 * a.nkv) * a.d)
        return Q3_ERR_BAD_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    if (f32) return f8 ? launch_append<float, true>(a, s) : launch_append<float, false>(a, s);
    return f8 ? launch_append<bf16, true>(a, s) : launch_append<bf16, false>(a, s);
}

template <typename T>
int read(const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, const int* page_table, int pages_per_seq,
         const int* seq_end, int n_seqs, int64_t n_pages, void* k_out, void* v_out, int out_pages, int nkv, int d, void* stream) {
    if (n_seqs <= 0 || out_pages <= 0) return 0;
    if (nkv <= 0 || d <= 0 || d > 256) return Q3_ERR_BAD_SIZE;
    if (n_seqs > 65535 || nkv > 65535) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch(read_kernel<T>, dim3(out_pages, nkv, n_seqs), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)k_pages,
                          (const uint8_t*)v_pages, (const uint8_t*)k_scales, (const uint8_t*)v_scales, page_table, pages_per_seq, seq_end,
                          n_pages, (T*)k_out, (T*)v_out, out_pages, nkv, d);
}

}  // namespace

Q3_EXPORT int q3_cache_append_f32(const void* qkv, void* q_out, void* k_pages, void* v_pages, void* k_scales, void* v_scales, const float* q_norm,
                                  const float* k_norm, const float* cos_tab, const float* sin_tab, float eps, const int* token_seq,
                                  const int* token_pos, const int* token_place, const int* page_table, int pages_per_seq, int64_t n_pages,
                                  int64_t n_tokens, int64_t row, int nq, int nkv, int d, int rotary_dim, int norm_once, void* stream) {
    return append({qkv, q_out, k_pages, v_pages, (uint8_t*)k_scales, (uint8_t*)v_scales, q_norm, k_norm, cos_tab, sin_tab, token_seq, token_pos,
                   token_place, page_table, pages_per_seq, nq, nkv, d, rotary_dim, norm_once, n_pages, n_tokens, row, eps},
                  true, k_scales != nullptr, stream);
}
Q3_EXPORT int q3_cache_append_bf16(const void* qkv, void* q_out, void* k_pages, void* v_pages, void* k_scales, void* v_scales, const float* q_norm,
                                   const float* k_norm, const float* cos_tab, const float* sin_tab, float eps, const int* token_seq,
                                   const int* token_pos, const int* token_place, const int* page_table, int pages_per_seq, int64_t n_pages,
                                   int64_t n_tokens, int64_t row, int nq, int nkv, int d, int rotary_dim, int norm_once, void* stream) {
    return append({qkv, q_out, k_pages, v_pages, (uint8_t*)k_scales, (uint8_t*)v_scales, q_norm, k_norm, cos_tab, sin_tab, token_seq, token_pos,
                   token_place, page_table, pages_per_seq, nq, nkv, d, rotary_dim, norm_once, n_pages, n_tokens, row, eps},
                  false, k_scales != nullptr, stream);
}

Q3_EXPORT int q3_cache_read_f32(const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, const int* page_table,
                                int pages_per_seq, const int* seq_end, int n_seqs, int64_t n_pages, void* k_out, void* v_out, int out_pages,
                                int nkv, int d, void* stream) {
    return read<float>(k_pages, v_pages, k_scales, v_scales, page_table, pages_per_seq, seq_end, n_seqs, n_pages, k_out, v_out, out_pages, nkv, d, stream);
}
Q3_EXPORT int q3_cache_read_bf16(const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales, const int* page_table,
                                 int pages_per_seq, const int* seq_end, int n_seqs, int64_t n_pages, void* k_out, void* v_out, int out_pages,
                                 int nkv, int d, void* stream) {
    return read<bf16>(k_pages, v_pages, k_scales, v_scales, page_table, pages_per_seq, seq_end, n_seqs, n_pages, k_out, v_out, out_pages, nkv, d, stream);
}

Q3_EXPORT int q3_cache_keep(void* store, void* scales, int64_t n_areas, int64_t n_pages, int nkv, int row_bytes, const int* page_table,
                            int pages_per_seq, const int* seq_pos0, const int* path, int path_len, int n_seqs, void* stream) {
    if (n_areas <= 0 || n_seqs <= 0 || path_len <= 0) return 0;
    if (nkv <= 0 || row_bytes <= 0) return Q3_ERR_BAD_SIZE;
    if (n_seqs > 65535 || n_areas > 0x7fffffff) return Q3_ERR_TOO_LARGE;
    if (row_bytes % 16 != 0 || !aligned16(store)) return Q3_ERR_MISALIGNED;
    return (int)q3_launch(keep_kernel, dim3((unsigned)n_areas, n_seqs), dim3(256), 0, (cudaStream_t)stream, (unsigned char*)store,
                          (uint8_t*)scales, n_pages, nkv, row_bytes, page_table, pages_per_seq, seq_pos0, path, path_len);
}
