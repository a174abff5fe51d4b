// Rows of the paged cache: written from a projection (normed, rotated, and quantised to 8 bits where the cache is kept so),
// read back, and moved after a step with drafted tokens.
//
// All three move bytes and compute next to nothing, so each is bound by memory; what each row costs:
//   append   reads (nq + 2 nkv) d values of the projection and d / 2 angles a token, writes nq d values and 2 nkv rows: 8,000 tokens of 32 + 16 heads of 128,
//            bfloat16 to 8 bits, 39.7 us (4.6 TB/s) where a normed value is rounded once, 44.8 with Qwen3's roundings after each step of the norm: the same
//            bytes, so instructions share the bound (the largest stall is memory all the same).  Into bfloat16 pages 41.4 and 43.8; 32-bit rows to 8 bits 62.6
//            (5.6 TB/s), as they are 68.4.  8 tokens 2.4 to 2.9;
//   read     reads d + 1 bytes a row and writes 2 d (bfloat16): 8 sequences of up to 8,000 rows and 8 heads of 128 in 43 us (6.0 TB/s), one of 2,000 3.7;
//            float32, 4 d written, 99 (4.3 TB/s);
//   keep     reads and writes the rows that move: 36 layers of 8 sequences 4.8 us, one sequence 3.5, which is a launch and a chain of three loads.
// Norm and rotation as in attention.cu's qkv_prepare (src/model/self_attention.cpp:122-152): y = x / sqrt(mean(x^2) + eps) w
// over a head, values i and i + r/2 of the first r turned by the angle of the token's position.  A token's place in the
// cache is given beside its position: drafted tokens of a tree stand side by side at places of their own, several at one position.
#include "../include/qwen3/cache_args.h"
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
            if (lane + 32 * t < d) to[lane + 32 * t] = (uint8_t)q3_codes2(make_float2(q3_is_number(y[t]) ? y[t] : __uint_as_float(0x7fffffffu), 0.0f), q3_exp2i(-k));
        if (lane == 0) (is_v ? a.v_scales : a.k_scales)[cell] = (uint8_t)(k + Q3_SCALE_BIAS);
    } else {
        T* to = (T*)(is_v ? a.v_pages : a.k_pages) + cell * d;
#pragma unroll
        for (int t = 0; t < PER; ++t)
            if (lane + 32 * t < d) to[lane + 32 * t] = from_f32<T>(y[t]);
    }
}

// ---- heads rotated whole or not at all, of a size that is made of packets: a group of L lanes a head, each lane with a packet of the first
// half and the one of the second half that it is turned with, so that a head's values are read once and in packets.
// A block takes 256 / L tokens and, one after the other, up to `per` heads of each: which kind of head it is at, its weights and all
// branches are the block's, a token's angles and page are looked up once, and the packets of the next head are asked for before the present one
// is worked on.  (Groups that each found their own head and token by a division spent 450 instructions a warp and turn, four times what the values need,
// and were bound by them: 8,000 tokens of 32 + 16 heads of 128 in 53 us.)  LANES 0: L as `lanes_log2` says.
template <typename T, bool F8, bool ONCE, int LANES>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a, int lanes_log2, int per) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int N = Pack<T>::N;
    const int lanes = LANES ? LANES : 1 << lanes_log2, l = threadIdx.x & (lanes - 1), d = a.d, half = d >> 1;
    const int tokens = LANES ? 256 / (LANES ? LANES : 1) : 256 >> lanes_log2;
    const int64_t n_raw = (int64_t)blockIdx.y * tokens + (LANES ? threadIdx.x / (LANES ? LANES : 1) : threadIdx.x >> lanes_log2);
    const bool mine = n_raw < a.n_tokens && (l * N < half);                  // (all lanes stay for the sums)
    const int64_t n = n_raw < a.n_tokens ? n_raw : 0;
    const int h0 = blockIdx.x * per, h1 = min(h0 + per, a.nq + 2 * a.nkv), i0 = mine ? l * N : 0;
    const T* src = (const T*)a.qkv + n * a.row + (int64_t)h0 * d + i0;
    Pack<T> x = load_pack<T>(src), y = load_pack<T>(src + half);
    float2 cs[N / 2], sn[N / 2];                   // pairs of values: the arithmetic takes two at once
    if (a.cos_tab != nullptr && h0 < a.nq + a.nkv) {
        const int64_t at = (int64_t)a.token_pos[n] * half + i0;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            const float4 c = *reinterpret_cast<const float4*>(a.cos_tab + at + e), s = *reinterpret_cast<const float4*>(a.sin_tab + at + e);
            cs[e / 2] = make_float2(c.x, c.y); cs[e / 2 + 1] = make_float2(c.z, c.w);
            sn[e / 2] = make_float2(s.x, s.y); sn[e / 2 + 1] = make_float2(s.z, s.w);
        }
    }
    int64_t page = 0;
    int at = 0;
    const bool has_place = h1 > a.nq && place_of(a.page_table, a.pages_per_seq, a.n_pages, a.token_seq[n], a.token_place[n], page, at) && mine;
    const float inv_d = 1.0f / (float)d;
    float2 wu[N / 2], wv[N / 2];
    const float* loaded = nullptr;                 // the weights that wu and wv hold
    for (int h = h0; h < h1; ++h) {
        const bool is_q = h < a.nq, is_v = h >= a.nq + a.nkv;
        const float* w = is_v ? nullptr : is_q ? a.q_norm : a.k_norm;
        float2 u[N / 2], v[N / 2];
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            u[e] = make_float2(x.get(2 * e), x.get(2 * e + 1));
            v[e] = make_float2(y.get(2 * e), y.get(2 * e + 1));
        }
        src += d;
        if (h + 1 < h1) {
            x = load_pack<T>(src);
            y = load_pack<T>(src + half);
        }
        if (w != nullptr) {
            if (w != loaded) {
                loaded = w;
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const float4 p = *reinterpret_cast<const float4*>(w + i0 + e), q = *reinterpret_cast<const float4*>(w + i0 + half + e);
                    wu[e / 2] = make_float2(p.x, p.y); wu[e / 2 + 1] = make_float2(p.z, p.w);
                    wv[e / 2] = make_float2(q.x, q.y); wv[e / 2 + 1] = make_float2(q.z, q.w);
                }
            }
            float2 sq = __fmul2_rn(u[0], u[0]);
#pragma unroll
            for (int e = 1; e < N / 2; ++e) sq = __ffma2_rn(u[e], u[e], sq);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) sq = __ffma2_rn(v[e], v[e], sq);
            float sum = (LANES ? (l * N < half) : mine) ? sq.x + sq.y : 0.0f;
#pragma unroll
            for (int o = (LANES ? LANES : 32) >> 1; o > 0; o >>= 1)
                if (LANES || o < lanes) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            const float inv = rsqrtf(sum * inv_d + a.eps);
            const float2 inv2 = make_float2(inv, inv);
            auto rounded = [](float2 z) { return ONCE ? z : make_float2(round_to<T>(z.x), round_to<T>(z.y)); };
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                u[e] = rounded(__fmul2_rn(rounded(__fmul2_rn(u[e], inv2)), wu[e]));
                v[e] = rounded(__fmul2_rn(rounded(__fmul2_rn(v[e], inv2)), wv[e]));
            }
        }
        if (!is_v && a.cos_tab != nullptr) {
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                const float2 p = u[e], q = v[e];
                u[e] = __ffma2_rn(q, make_float2(-sn[e].x, -sn[e].y), __fmul2_rn(p, cs[e]));
                v[e] = __ffma2_rn(p, sn[e], __fmul2_rn(q, cs[e]));
            }
        }
        if (is_q || !F8) {
            const int64_t cell = (page * a.nkv + (is_v ? h - a.nq - a.nkv : h - a.nq)) * PAGE + at;
            T* to = is_q ? (T*)a.q_out + (n * a.nq + h) * d + i0 : (T*)(is_v ? a.v_pages : a.k_pages) + cell * d + i0;
            if (is_q ? mine : has_place) {
                Pack<T> p, q;
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    p.set(2 * e, u[e].x);
                    p.set(2 * e + 1, u[e].y);
                    q.set(2 * e, v[e].x);
                    q.set(2 * e + 1, v[e].y);
                }
                store_pack<T>(to, p);
                store_pack<T>(to + half, q);
            }
            continue;
        }
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            if (!ONCE) {
                u[e] = make_float2(round_to<T>(u[e].x), round_to<T>(u[e].y));
                v[e] = make_float2(round_to<T>(v[e].x), round_to<T>(v[e].y));
            }
            top = fmaxf(top, fmaxf(fmaxf(fabsf(u[e].x), fabsf(u[e].y)), fmaxf(fabsf(v[e].x), fabsf(v[e].y))));       // (passes over NaN)
        }
        auto of_head = [&](float z) {
            z = (LANES ? (l * N < half) : mine) ? z : 0.0f;
#pragma unroll
            for (int o = (LANES ? LANES : 32) >> 1; o > 0; o >>= 1)
                if (LANES || o < lanes) z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, o));
            return z;
        };
        top = of_head(top);
        if (__any_sync(0xffffffffu, !q3_is_number(top))) {                       // infinities become NaN, and do not count
            const float nan = __uint_as_float(0x7fffffffu);
            top = 0.0f;
#pragma unroll
            for (int e = 0; e < N / 2; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float& z = i == 0 ? u[e].x : i == 1 ? u[e].y : i == 2 ? v[e].x : v[e].y;
                    if (!q3_is_number(z)) z = nan;
                    top = fmaxf(top, fabsf(z));
                }
            top = of_head(top);
        }
        if (has_place) {
            const int64_t cell = (page * a.nkv + (is_v ? h - a.nq - a.nkv : h - a.nq)) * PAGE + at;
            const int exponent = q3_scale_exponent(top);
            const float inv = q3_exp2i(-exponent);
            uint8_t* to = (uint8_t*)(is_v ? a.v_pages : a.k_pages) + cell * d + i0;
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                const float2* z = side ? v : u;
                uint32_t c[N / 4];
#pragma unroll
                for (int e = 0; e < N / 4; ++e) c[e] = q3_codes2(z[2 * e], inv) | q3_codes2(z[2 * e + 1], inv) << 16;
                if constexpr (N == 8) *reinterpret_cast<uint2*>(to + side * half) = make_uint2(c[0], c[1]);
                else *reinterpret_cast<uint32_t*>(to + side * half) = c[0];
            }
            if (l == 0) (is_v ? a.v_scales : a.k_scales)[cell] = (uint8_t)(exponent + Q3_SCALE_BIAS);
        }
    }
}

template <typename T, bool F8, bool ONCE>
cudaError_t launch_append_packets(const AppendArgs& a, int log2, int per, cudaStream_t stream) {
    const int tokens = 256 >> log2;
    const dim3 grid((a.nq + 2 * a.nkv + per - 1) / per, (unsigned)((a.n_tokens + tokens - 1) / tokens));
    auto kernel = log2 == 2 ? append_kernel<T, F8, ONCE, 4> : log2 == 3 ? append_kernel<T, F8, ONCE, 8> : log2 == 4 ? append_kernel<T, F8, ONCE, 16>
                                                                                                                  : append_kernel<T, F8, ONCE, 0>;
    return q3_launch(kernel, grid, dim3(256), 0, stream, a, log2, per);
}

template <typename T, bool F8>
int launch_append(const AppendArgs& a, cudaStream_t stream) {
    constexpr int N = Pack<T>::N;
    const int64_t vecs = a.n_tokens * (a.nq + 2 * a.nkv);
    auto whole = [](const void* p) { return p == nullptr || aligned16(p); };
    // packets: 16 bytes of both halves of a head wherever it begins, and of its weights and angles (codes: N bytes)
    const bool packets = a.d % (2 * N) == 0 && (a.rot == a.d || a.cos_tab == nullptr) && a.row % N == 0 && whole(a.qkv) && whole(a.q_out) && whole(a.k_pages) &&
                         whole(a.v_pages) && whole(a.q_norm) && whole(a.k_norm) && whole(a.cos_tab) && whole(a.sin_tab);
    if (packets) {
        int log2 = 0;
        while ((N << log2) < a.d / 2) ++log2;
        const int tokens = 256 >> log2;
        if ((a.n_tokens + tokens - 1) / tokens > 65535) return Q3_ERR_TOO_LARGE;
        // four heads a block once that leaves more blocks than an SM and a half (700 tokens of 48 heads of 128: 5.3 us against 6.4 with one, 200: 4.5 / 3.4,
        // 8,000: 40 / 62)
        const int per = ((a.n_tokens + tokens - 1) / tokens) * (a.nq + 2 * a.nkv) > 6 * (int64_t)q3_device_sm_count() ? 4 : 1;
        return (int)(a.norm_once ? launch_append_packets<T, F8, true>(a, log2, per, stream) : launch_append_packets<T, F8, false>(a, log2, per, stream));
    }
    const int64_t blocks = (vecs + 7) / 8;
    if (blocks > 0x7fffffff) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch(append_any_kernel<T, F8>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
}

// ---- the cached rows of sequences as pages of T, page j of sequence s at s * out_pages + j
template <typename T>
__global__ void __launch_bounds__(256)
read_kernel(const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const uint8_t* __restrict__ k_scales,
            const uint8_t* __restrict__ v_scales, const int* __restrict__ page_table, int pages_per_seq, const int* __restrict__ seq_end,
            int64_t n_pages, T* __restrict__ k_out, T* __restrict__ v_out, int out_pages, int nkv, int d, bool packets) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.z, j = blockIdx.x, g = blockIdx.y, live = min(PAGE, seq_end[seq] - j * PAGE);
    if (live <= 0 || j >= pages_per_seq) return;
    const int64_t page = page_table[(int64_t)seq * pages_per_seq + j];
    if (page < 0 || page >= n_pages) return;
    const int64_t from = (page * nkv + g) * PAGE, to = (((int64_t)seq * out_pages + j) * nkv + g) * PAGE;
    if (packets) {
        // eight codes a turn, keys and values, all of a thread's copies asked for before the first is used
        constexpr int TURNS = 4;
        const int per_row = d / 8, n = PAGE * per_row;
        for (int i0 = threadIdx.x; i0 < n; i0 += blockDim.x * TURNS) {
            uint2 codes[2][TURNS];
            uint8_t scale[2][TURNS];
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const int i = i0 + u * blockDim.x;
                if (i < n) {
                    codes[0][u] = reinterpret_cast<const uint2*>(k_pages + from * d)[i];
                    codes[1][u] = reinterpret_cast<const uint2*>(v_pages + from * d)[i];
                    scale[0][u] = k_scales[from + i / per_row];
                    scale[1][u] = v_scales[from + i / per_row];
                }
            }
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const int i = i0 + u * blockDim.x;
                if (i >= n) break;
#pragma unroll
                for (int side = 0; side < 2; ++side) {
                    const float s = q3_exp2i((int)scale[side][u] - Q3_SCALE_BIAS);
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 two = __half22float2(q3_half2_of((e < 2 ? codes[side][u].x : codes[side][u].y) >> (16 * (e & 1))));
                        v[2 * e] = i / per_row < live ? two.x * s : 0.0f;
                        v[2 * e + 1] = i / per_row < live ? two.y * s : 0.0f;
                    }
                    T* out = (side ? v_out : k_out) + to * d + 8 * (int64_t)i;
#pragma unroll
                    for (int e = 0; e < 8; e += Pack<T>::N) {
                        Pack<T> p;
#pragma unroll
                        for (int k = 0; k < Pack<T>::N; ++k) p.set(k, v[e + k]);
                        store_pack<T>(out + e, p);
                    }
                }
            }
        }
        return;
    }
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
    constexpr int TURNS = 4;
    const int pos0 = seq_pos0[seq];
    for (int i = threadIdx.x; i < nkv * per_head; i += blockDim.x) {
        const int g = i / per_head, c = i % per_head;
        for (int n0 = 0; n0 < path_len; n0 += TURNS) {                  // (a row of the path that a turn writes over was read in this turn or before)
            uint4 rows[TURNS];
            int64_t to[TURNS];
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                to[u] = -1;
                const int n = n0 + u, node = n < path_len ? path[(int64_t)seq * path_len + n] : -1;
                int64_t from_page, to_page;
                int from_at, to_at;
                if (node <= n || !place_of(page_table, pages_per_seq, n_pages, seq, pos0 + node, from_page, from_at) ||
                    !place_of(page_table, pages_per_seq, n_pages, seq, pos0 + n, to_page, to_at))
                    continue;
                const int64_t from = ((area * n_pages + from_page) * nkv + g) * PAGE + from_at;
                to[u] = ((area * n_pages + to_page) * nkv + g) * PAGE + to_at;
                if (c == packets) rows[u].x = scales[from];
                else rows[u] = *reinterpret_cast<const uint4*>(store + from * row_bytes + c * 16);
            }
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                if (to[u] < 0) continue;
                if (c == packets) scales[to[u]] = (uint8_t)rows[u].x;
                else *reinterpret_cast<uint4*>(store + to[u] * row_bytes + c * 16) = rows[u];
            }
        }
    }
}

int append(const q3_cache_append_args& x, bool f32) {
    const AppendArgs a = {x.qkv, x.q_out, x.k_pages, x.v_pages, (uint8_t*)x.k_scales, (uint8_t*)x.v_scales, (const float*)x.q_norm, (const float*)x.k_norm,
                          (const float*)x.cos_tab, (const float*)x.sin_tab, (const int*)x.token_seq, (const int*)x.token_pos, (const int*)x.token_place,
                          (const int*)x.page_table, x.pages_per_seq, x.nq, x.nkv, x.d, x.rotary_dim, x.norm_once, x.n_pages, x.n_tokens, x.row, (float)x.eps};
    if (a.n_tokens <= 0) return 0;
    if (a.nq <= 0 || a.nkv <= 0 || a.d <= 0 || a.d > 256 || a.rot < 0 || a.rot > a.d || (a.rot & 1) || a.row < (int64_t)(a.nq + 2 * a.nkv) * a.d)
        return Q3_ERR_BAD_SIZE;
    cudaStream_t s = (cudaStream_t)x.stream;
    const bool f8 = a.k_scales != nullptr;
    if (f32) return f8 ? launch_append<float, true>(a, s) : launch_append<float, false>(a, s);
    return f8 ? launch_append<bf16, true>(a, s) : launch_append<bf16, false>(a, s);
}

template <typename T> int read(const q3_cache_read_args& x) {
    if (x.n_seqs <= 0 || x.out_pages <= 0) return 0;
    if (x.nkv <= 0 || x.d <= 0 || x.d > 256) return Q3_ERR_BAD_SIZE;
    if (x.n_seqs > 65535 || x.nkv > 65535) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch(read_kernel<T>, dim3(x.out_pages, x.nkv, x.n_seqs), dim3(256), 0, (cudaStream_t)x.stream, (const uint8_t*)x.k_pages,
                          (const uint8_t*)x.v_pages, (const uint8_t*)x.k_scales, (const uint8_t*)x.v_scales, (const int*)x.page_table, x.pages_per_seq,
                          (const int*)x.seq_end, x.n_pages, (T*)x.k_out, (T*)x.v_out, x.out_pages, x.nkv, x.d,
                          x.d % 8 == 0 && aligned16(x.k_pages) && aligned16(x.v_pages) && aligned16(x.k_out) && aligned16(x.v_out));
}

}  // namespace

Q3_EXPORT int q3_cache_append_f32(const q3_cache_append_args* a) { return append(*a, true); }
Q3_EXPORT int q3_cache_append_bf16(const q3_cache_append_args* a) { return append(*a, false); }
Q3_EXPORT int q3_cache_read_f32(const q3_cache_read_args* a) { return read<float>(*a); }
Q3_EXPORT int q3_cache_read_bf16(const q3_cache_read_args* a) { return read<bf16>(*a); }

Q3_EXPORT int q3_cache_keep(const q3_cache_keep_args* a) {
    if (a->n_areas <= 0 || a->n_seqs <= 0 || a->path_len <= 0) return 0;
    if (a->nkv <= 0 || a->row_bytes <= 0) return Q3_ERR_BAD_SIZE;
    if (a->n_seqs > 65535 || a->n_areas > 0x7fffffff) return Q3_ERR_TOO_LARGE;
    if (a->row_bytes % 16 != 0 || !aligned16(a->store)) return Q3_ERR_MISALIGNED;
    return (int)q3_launch(keep_kernel, dim3((unsigned)a->n_areas, a->n_seqs), dim3(256), 0, (cudaStream_t)a->stream, (unsigned char*)a->store,
                          (uint8_t*)a->scales, a->n_pages, a->nkv, a->row_bytes, (const int*)a->page_table, a->pages_per_seq, (const int*)a->seq_pos0,
                          (const int*)a->path, a->path_len);
}
