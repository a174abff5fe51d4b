// Products of 8-bit integers with a scale for each token and channel: y[m, n] = (sum_k x[m, k] w[n, k]) sx[m] sw[n].
//
// The sum is taken in whole numbers, which 32 bits hold for K up to 131,071 (2^31 / 2^14), so it does not hang on the order: every form below gives
// the same bits for a token, whatever the batch around it.  It becomes a 32-bit float, is scaled by the token's and then by the channel's scale and
// rounded to the output type.  With a gate, gate and up stay in 32 bits until their product is rounded.
#include "common.cuh"
#include "../include/qwen3/int8_args.h"

namespace {

template <typename OutT> __device__ __forceinline__ OutT to_out(float v);
template <> __device__ __forceinline__ float to_out<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 to_out<bf16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float scaled(int sum, float token, float channel) { return (float)sum * token * channel; }

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
    uint4 v;   // not volatile: the compiler may hoist and batch these loads
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct Product {
    const int8_t *x, *w;
    const float *sx, *sw;
    void* y;
    int64_t ldx, ldw;
    int M, N, K;
};

// ---------------------------------------------------------------------------------------------
// Few tokens: bound by reading W once.  A block owns 16 rows of W and shares K among its warps; a lane reads 16 consecutive bytes of two rows of W a
// step and hands them to mma.m16n8k32 as they come, as the 16-row operand, with eight tokens as the columns: a sum over k does not care about the
// order of k, so the token's 16 bytes at the same place are the other operand, and nothing is shuffled or staged.  Grid (16 rows of W, 8 * MT tokens).
template <int MT, int WARPS, int PF, int MINB, int GATED, typename OutT>
__global__ void __launch_bounds__(WARPS * 32, MINB) few_kernel(const Product p) {
    extern __shared__ __align__(16) int red[];   // [WARPS][8 * MT][17]
    constexpr int COLS = 8 * MT, LD = 17;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, tq = lane & 3;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * COLS;
    const int nkb = (p.K + 63) >> 6;                           // K in steps of 64: 16 bytes a lane of a row's four
    const int kb_begin = (int)(((int64_t)warp * nkb) / WARPS), kb_end = (int)(((int64_t)(warp + 1) * nkb) / WARPS);

    int acc[MT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0;
    const int8_t* wrow[2];
    bool wok[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = n0 + h * 8 + quad;
        wok[h] = n < p.N;
        wrow[h] = p.w + (int64_t)(wok[h] ? n : 0) * p.ldw + tq * 16;
    }
    const int8_t* xrow[MT];
    bool xok[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int row = m0 + m * 8 + quad;
        xok[m] = row < p.M;
        xrow[m] = p.x + (int64_t)(xok[m] ? row : 0) * p.ldx + tq * 16;
    }
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 w[PF][2], x[PF][MT];
    // a packet that begins inside the row may be read whole (rows are a multiple of 16 bytes apart); what lies behind the row counts nothing,
    // because the tokens' bytes there are taken as zeros
    auto load_w = [&](int s, int kb) {
        const int k = kb * 64;
        const bool in = kb < kb_end && k + tq * 16 < p.K;
#pragma unroll
        for (int h = 0; h < 2; ++h) w[s][h] = in && wok[h] ? ld_stream16(wrow[h] + k) : zero;
    };
    auto load_x = [&](int s, int kb) {
        const int k = kb * 64, left = p.K - k - tq * 16;
        const bool in = kb < kb_end && left > 0;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            x[s][m] = in && xok[m] ? *reinterpret_cast<const uint4*>(xrow[m] + k) : zero;
            if (in && left < 16) {
                uint32_t* v = &x[s][m].x;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] &= left >= 4 * i + 4 ? 0xffffffffu : left <= 4 * i ? 0u : (1u << (8 * (left - 4 * i))) - 1u;
            }
        }
    };
#pragma unroll
    for (int s = 0; s < PF; ++s) load_w(s, kb_begin + s);
    pdl_wait();
#pragma unroll
    for (int s = 0; s < PF; ++s) load_x(s, kb_begin + s);
    for (int kb = kb_begin; kb < kb_end; kb += PF) {
#pragma unroll
        for (int s = 0; s < PF; ++s) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                mma_s8(acc[m], w[s][0].x, w[s][1].x, w[s][0].y, w[s][1].y, x[s][m].x, x[s][m].y);
                mma_s8(acc[m], w[s][0].z, w[s][1].z, w[s][0].w, w[s][1].w, x[s][m].z, x[s][m].w);
            }
            load_w(s, kb + s + PF);      // steps past the end load zeros, which add nothing
            load_x(s, kb + s + PF);
        }
    }
    pdl_launch_dependents();

    int* mine = red + warp * COLS * LD;  // accumulator (row n = quad [+ 8], token 2 tq [+ 1]) -> [warp][token][row]
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int c = m * 8 + tq * 2;
        mine[c * LD + quad] = acc[m][0];
        mine[(c + 1) * LD + quad] = acc[m][1];
        mine[c * LD + quad + 8] = acc[m][2];
        mine[(c + 1) * LD + quad + 8] = acc[m][3];
    }
    __syncthreads();
    auto total = [&](int m, int n) {
        int sum = 0;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) sum += red[(v * COLS + m) * LD + n];
        return sum;
    };
    if constexpr (GATED == 0) {
        for (int idx = threadIdx.x; idx < 16 * COLS; idx += WARPS * 32) {
            const int n = idx % 16, m = idx / 16;
            if (m0 + m >= p.M || n0 + n >= p.N) continue;
            ((OutT*)p.y)[(int64_t)(m0 + m) * p.N + n0 + n] = to_out<OutT>(scaled(total(m, n), p.sx[m0 + m], p.sw[n0 + n]));
        }
    } else {
        for (int idx = threadIdx.x; idx < 8 * COLS; idx += WARPS * 32) {
            const int n = idx % 8, m = idx / 8;
            if (m0 + m >= p.M || n0 + n >= p.N) continue;
            const float sx = p.sx[m0 + m];
            const float g = scaled(total(m, n), sx, p.sw[n0 + n]), u = scaled(total(m, n + 8), sx, p.sw[n0 + n + 8]);
            ((OutT*)p.y)[(int64_t)(m0 + m) * (p.N >> 1) + (n0 >> 1) + n] = to_out<OutT>(gate_activation<GATED>(g) * u);
        }
    }
}

template <int MT, int WARPS, int PF, int MINB, int GATED, typename OutT> int launch_few(const Product& p, cudaStream_t stream) {
    const int64_t tokens = (p.M + 8 * MT - 1) / (8 * MT);
    if (tokens > 65535) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch(few_kernel<MT, WARPS, PF, MINB, GATED, OutT>, dim3((unsigned)((p.N + 15) / 16), (unsigned)tokens), dim3(WARPS * 32),
                          WARPS * 8 * MT * 17 * 4, stream, p);
}

template <int GATED, typename OutT> int few(const Product& p, cudaStream_t stream) {
    return launch_few<1, 8, 4, 3, GATED, OutT>(p, stream);
}

int product_of(const q3_gemm_int8_args& a, Product& p) {
    if (a.width <= 0 || a.width > 131071 || a.activation < 0 || a.activation > 2 || (a.activation != 0 && a.channels % 16 != 0)) return Q3_ERR_BAD_SIZE;
    if (a.x_stride < a.width || a.w_stride < a.width) return Q3_ERR_BAD_SIZE;
    if (!aligned16(a.x) || !aligned16(a.w) || a.x_stride % 16 != 0 || a.w_stride % 16 != 0) return Q3_ERR_MISALIGNED;
    p = Product{(const int8_t*)a.x, (const int8_t*)a.w, (const float*)a.x_scales, (const float*)a.w_scales, a.y, a.x_stride, a.w_stride,
                a.rows, a.channels, a.width};
    return 0;
}

#define Q3_BY_EPILOGUE(CALL)                                                                      \
    do {                                                                                          \
        if (a->activation == 1) return a->out_is_f32 ? CALL(1, float) : CALL(1, bf16);             \
        if (a->activation == 2) return a->out_is_f32 ? CALL(2, float) : CALL(2, bf16);             \
        return a->out_is_f32 ? CALL(0, float) : CALL(0, bf16);                                     \
    } while (0)

}  // namespace

// Few tokens, W streamed (any number of tokens is taken; W is read once for every eight).
Q3_EXPORT int q3_gemm_int8_few(const q3_gemm_int8_args* a) {
    if (a->rows <= 0 || a->channels <= 0) return 0;
    Product p;
    const int bad = product_of(*a, p);
    if (bad) return bad;
#define Q3_FEW(G, T) few<G, T>(p, (cudaStream_t)a->stream)
    Q3_BY_EPILOGUE(Q3_FEW);
#undef Q3_FEW
}
