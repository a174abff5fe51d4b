// Products of 8-bit integers with a scale for each token and channel: y[m, n] = (sum_k x[m, k] w[n, k]) sx[m] sw[n].
//
// The sum is taken in whole numbers, which 32 bits hold for K up to 131,071 (2^31 / 2^14), so it does not hang on the order: every form below gives
// the same bits for a token, whatever the batch around it.  It becomes a 32-bit float, is scaled by the token's and then by the channel's scale and
// rounded to the output type.  With a gate, gate and up stay in 32 bits until their product is rounded.
//
// Three forms: few tokens on mma.sync, W streamed through registers; up to some hundred on tcgen05 with W as the 128-row operand and K split over a
// cluster; prompts on pairs of SMs.  A row of codes is 128 bytes of K a step, one swizzle row, and an instruction takes 32 of them.  Every wait on an
// mbarrier is bounded: after Q3_WAIT_LIMIT polls the thread records where it gave up in `status` and the block winds down (tensor memory is
// freed on every path, and the cluster barriers are reached by every thread on every path).
#include <cuda.h>

#include "common.cuh"
#include "tcgen05.cuh"
#include "tcgen05_pair.cuh"
#include "tma.cuh"
#include "../include/qwen3/int8_args.h"

namespace {

template <typename OutT> __device__ __forceinline__ OutT to_out(float v);
template <> __device__ __forceinline__ float to_out<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16 to_out<bf16>(float v) { return __float2bfloat16_rn(v); }

// The activation of a value whose product with `up` is rounded to OutT.
template <int GATED, typename OutT> __device__ __forceinline__ float activated(float z) {
    if constexpr (GATED == 1) return silu_for<OutT>(z);
    return gate_activation<GATED>(z);
}

__device__ __forceinline__ float scaled(int sum, float token, float channel) { return (float)sum * token * channel; }

// Read once, past the L1.  W may have been written by the kernel ahead, which a dependent launch overlaps: so the load is neither one of memory that
// stays as it is for the whole kernel (.nc), nor may it be moved over the wait for that kernel (volatile, with its memory).
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

inline int most(int a, int b) { return a > b ? a : b; }
constexpr int GRID_YZ = 65535;         // blocks along a grid's second and third axis

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
    pdl_wait();                          // (for W, too: the caller may just have quantised it)
#pragma unroll
    for (int s = 0; s < PF; ++s) load_w(s, kb_begin + s);
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
            ((OutT*)p.y)[(int64_t)(m0 + m) * (p.N >> 1) + (n0 >> 1) + n] = to_out<OutT>(activated<GATED, OutT>(g) * u);
        }
    }
}

template <int MT, int WARPS, int PF, int MINB, int GATED, typename OutT> int launch_few(const Product& p, cudaStream_t stream) {
    const int64_t tokens = (p.M + 8 * MT - 1) / (8 * MT);
    if (tokens > GRID_YZ) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch(few_kernel<MT, WARPS, PF, MINB, GATED, OutT>, dim3((unsigned)((p.N + 15) / 16), (unsigned)tokens), dim3(WARPS * 32),
                          WARPS * 8 * MT * 17 * 4, stream, p);
}

// Warps that share K, steps in flight and blocks an SM.  Up to eight tokens (16 warps, 2 steps, 2 blocks / 8, 4, 3 / 8, 2, 4, us): as long as all blocks
// run at once, more warps (4,096 x 4,096 4.9 / 5.6 / 5.6, 4,096 x 12,288 10.1 / 11.2 / 12.8), then more steps where K is long (5,120 x 17,408 21.6 /
// 16.7 / 18.9), else more blocks (6,144 x 4,096 7.3 / 6.6 / 6.1, gated 24,576 x 4,096 21.1 / 19.5 / 18.2).
template <int GATED, typename OutT> int few(const Product& p, cudaStream_t stream) {
    const int sms = q3_device_sm_count(), blocks = (p.N + 15) / 16;
    if (p.M <= 8) {
        if (blocks <= 2 * sms) return launch_few<1, 16, 2, 2, GATED, OutT>(p, stream);
        if (blocks <= 3 * sms && p.K >= 8192) return launch_few<1, 8, 4, 3, GATED, OutT>(p, stream);
        return launch_few<1, 8, 2, 4, GATED, OutT>(p, stream);
    }
    if (p.M <= 16)
        return blocks <= 2 * sms ? launch_few<2, 16, 1, 2, GATED, OutT>(p, stream) : launch_few<2, 8, 2, 3, GATED, OutT>(p, stream);
    return launch_few<4, 8, 2, 2, GATED, OutT>(p, stream);
}

// ---------------------------------------------------------------------------------------------
// Up to some hundred tokens, weights first: D[128 rows of W, MT tokens] = W tile . X tile^T on tcgen05, so that the 128-row operand is full whatever
// the number of tokens.  Where W has few rows, K is split over the blocks of a cluster; their partial tiles meet in shared memory, and each block
// adds up, scales and writes a share of the tokens.  Grid (tiles of 128 rows of W, K ranges, tiles of MT tokens), clusters (1, K ranges, 1).
//   warp 0     TMA producer
//   warp 1     allocates tensor memory; one elected thread issues the products and hands each stage back to the producer
//   warps 2-9  bring the accumulator (a row of W a thread, every other 16 tokens) into shared memory, and the scales
constexpr int BM = 128, BK = 128, UMMA_K = 32;
constexpr int MID_SETS = 2, THREADS = 64 + 128 * MID_SETS;    // drain warps: twice the four quarters of tensor memory
constexpr int PART_LD = BM + 4;         // words per token of the partial tile (rows stay 16-byte aligned)

__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ int4 ld_cluster_i4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
template <typename OutT> __device__ __forceinline__ void store4(OutT* p, const float (&v)[4], bool whole, int valid) {
    if (whole && valid >= 4) {
        if constexpr (sizeof(OutT) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
            *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < valid) p[i] = to_out<OutT>(v[i]);
}

// A producer's end: the copies of its `issued` steps have landed and been read (every stage has been handed back), or the limit has run out.  No block goes
// while its copies are under way, also where another role has given up; otherwise the accumulator that its last warps wait for is later than this.
template <int STAGES> __device__ __forceinline__ void wait_for_stages(uint32_t empty, uint32_t issued) {
    for (uint32_t i = issued; i < issued + STAGES; ++i) mbar_wait(empty + i % STAGES * 8, ((i / STAGES) & 1u) ^ 1u);
}

template <int MT, int STAGES, int MINB, int GATED, typename OutT>
__global__ void __launch_bounds__(THREADS, MINB)
mid_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Product p, int* __restrict__ status) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ float channel_scales[BM], token_scales[MT];
    constexpr int A_BYTES = BM * BK, B_BYTES = MT * BK, STAGE_BYTES = A_BYTES + B_BYTES;   // multiples of 1024
    constexpr uint32_t TMEM_COLS = MT < 32 ? 32 : MT;
    static_assert(MT == 16 || (MT % 32 == 0 && MT <= 256), "token tile: the N of an M = 128 product of 8-bit integers");
    // the partial tile reuses the stages (and what lies behind them, if it is the larger of the two)
    constexpr int RING_BYTES = STAGES * STAGE_BYTES > MT * PART_LD * 4 ? STAGES * STAGE_BYTES : (MT * PART_LD * 4 + 1023) / 1024 * 1024;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;         // 128-byte swizzle wants 1024-byte tiles
    const uint32_t bars = base + RING_BYTES;                              // full[STAGES], empty[STAGES], done, tmem slot
    const uint32_t bar_done = bars + 2 * STAGES * 8, tmem_slot = bar_done + 8;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * BM, m0 = blockIdx.z * MT;
    const uint32_t rank = cluster_rank(), ranks = gridDim.y;
    const int nkb_all = (p.K + BK - 1) / BK;
    const int kb_begin = (int)(((int64_t)rank * nkb_all) / ranks), kb_end = (int)(((int64_t)(rank + 1) * nkb_all) / ranks);
    const int nkb = kb_end - kb_begin;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bars + s * 8, 1);
            mbar_init(bars + (STAGES + s) * 8, 1);
        }
        mbar_init(bar_done, 1);
        mbar_init_fence();
    }
    __syncthreads();
    // the producer starts its stream now; tensor memory is handed out meanwhile and its address goes to the warps that use it
    uint32_t tmem_base = 0;
    if (warp >= 1) {
        if (warp == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
        asm volatile("bar.sync 1, %0;" ::"n"(THREADS - 32) : "memory");
        tc_fence_after();
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    }

    if (warp == 0) {
        if (lane == 0) {
            pdl_wait();              // (for W, too: the caller may just have quantised it; asking for it earlier gained nothing to 4 %)
            int i = 0;
            for (; i < nkb; ++i) {
                const int s = i % STAGES;
                if (!mbar_wait(bars + (STAGES + s) * 8, ((uint32_t)(i / STAGES) & 1u) ^ 1u)) {      // the stage is free
                    atomicExch(status, 1);
                    break;
                }
                const uint32_t a = base + s * STAGE_BYTES, b = a + A_BYTES;
                mbar_expect_tx(bars + s * 8, STAGE_BYTES);
                tma_load_2d(a, &map_w, bars + s * 8, (kb_begin + i) * BK, n0);
                tma_load_2d(b, &map_x, bars + s * 8, (kb_begin + i) * BK, m0);
            }
            wait_for_stages<STAGES>(bars + STAGES * 8, (uint32_t)i);
        }
    } else if (warp == 1) {
        // the whole warp walks the K steps and one elected thread issues, so that descriptors stay in uniform registers
        constexpr uint32_t idesc = make_idesc_i8(BM, MT);
        const uint64_t desc0 = desc_k_major(base);
        const uint32_t acc = __shfl_sync(0xffffffffu, tmem_base, 0);
        for (int i = 0; i < nkb; ++i) {
            const uint32_t s = (uint32_t)i % STAGES;
            if (!mbar_wait_warp(bars + s * 8, ((uint32_t)i / STAGES) & 1u)) {    // the tiles have landed
                if (lane == 0) atomicExch(status, 2);
                break;
            }
            tc_fence_after();
            const uint64_t da = desc0 + (uint64_t)(s * (STAGE_BYTES >> 4)), db = da + (A_BYTES >> 4);
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k)                        // 32 bytes further along K per step
                    tc_mma_i8(acc, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, (i > 0 || k > 0) ? 1u : 0u);
                tc_commit(bars + (STAGES + s) * 8);                          // frees the stage when the products are done
            }
            __syncwarp();
        }
        if (elect_one()) tc_commit(bar_done);                                // accumulator complete (or abandoned)
        __syncwarp();
    } else {
        // warps own lanes 32 * (warp % 4) .. of tensor memory: accumulator -> part[token][row of W].  The scales are there before they are needed: fetched
        // in the end they are the longest step of it.
        const int t = threadIdx.x - 64;
        pdl_wait();
        if (t < BM) channel_scales[t] = n0 + t < p.N ? p.sw[n0 + t] : 0.0f;
        if (t < MT) token_scales[t] = m0 + t < p.M ? p.sx[m0 + t] : 0.0f;
        const bool ok = mbar_wait(bar_done, 0);                              // every load has landed and been consumed,
        if (!ok && lane == 0) atomicExch(status, 3);                         // so the stages may be overwritten
        tc_fence_after();
        uint32_t* part = reinterpret_cast<uint32_t*>(smem_raw + (base - smem_u32(smem_raw)));
        const int lane_base = (warp & 3) * 32;
#pragma unroll 1
        for (int c = 16 * ((warp - 2) >> 2); c < MT; c += 16 * MID_SETS) {
            uint32_t r[16];
            if (ok && nkb > 0) {
                tc_ld16(tmem_base + ((uint32_t)lane_base << 16) + (uint32_t)c, r);
                tc_wait_ld();
            } else {                                                          // an empty K range adds nothing
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = 0u;
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) part[(c + j) * PART_LD + lane_base + lane] = r[j];
        }
    }
    tc_fence_before();
    __syncwarp();
    if (ranks > 1) cluster_sync();                                            // every block's partial tile is in place
    else __syncthreads();                                                     // (a block on its own: its own tile)

    pdl_wait();                                                               // no global write before this
    {
        // this block finishes the tokens m with m % ranks == rank
        OutT* Y = (OutT*)p.y;
        const int out_n = GATED ? (p.N >> 1) : p.N;
        const bool whole = (out_n % 4 == 0) && ((reinterpret_cast<uintptr_t>(Y) & 15u) == 0);
        constexpr int GROUPS = GATED ? 16 : 32;                               // groups of four outputs per token and tile
        const int my_tokens = (MT - (int)rank + (int)ranks - 1) / (int)ranks;
        auto sum4 = [&](uint32_t addr) {                                      // all blocks' parts are asked for together
            int4 v[8];
#pragma unroll
            for (uint32_t s = 0; s < 8; ++s) v[s] = s < ranks ? ld_cluster_i4(map_to_rank(addr, s)) : make_int4(0, 0, 0, 0);
            int4 sum = v[0];
#pragma unroll
            for (int s = 1; s < 8; ++s) { sum.x += v[s].x; sum.y += v[s].y; sum.z += v[s].z; sum.w += v[s].w; }
            return sum;
        };
        for (int idx = threadIdx.x; idx < my_tokens * GROUPS; idx += THREADS) {
            const int local = (idx / GROUPS) * (int)ranks + (int)rank, g = idx % GROUPS;
            const int m = m0 + local;
            if (m >= p.M) continue;
            const float sx = token_scales[local];
            if constexpr (GATED == 0) {
                const int n = n0 + 4 * g;
                if (n >= p.N) continue;
                const int4 sum = sum4(base + (uint32_t)(local * PART_LD + 4 * g) * 4u);
                const float* sw = channel_scales + 4 * g;
                const float v[4] = {scaled(sum.x, sx, sw[0]), scaled(sum.y, sx, sw[1]), scaled(sum.z, sx, sw[2]), scaled(sum.w, sx, sw[3])};
                store4<OutT>(Y + (int64_t)m * p.N + n, v, whole, p.N - n);
            } else {
                // rows 16t + 4h .. + 3 are gates, rows 16t + 8 + 4h .. + 3 the ups of features 8t + 4h .. + 3
                const int t = g >> 1, h = g & 1, n = n0 + 16 * t + 4 * h;
                if (n >= p.N) continue;
                const uint32_t addr = base + (uint32_t)(local * PART_LD + 16 * t + 4 * h) * 4u;
                const int4 gs = sum4(addr), us = sum4(addr + 32u);
                const float* sw = channel_scales + 16 * t + 4 * h;
                const float v[4] = {activated<GATED, OutT>(scaled(gs.x, sx, sw[0])) * scaled(us.x, sx, sw[8]),
                                    activated<GATED, OutT>(scaled(gs.y, sx, sw[1])) * scaled(us.y, sx, sw[9]),
                                    activated<GATED, OutT>(scaled(gs.z, sx, sw[2])) * scaled(us.z, sx, sw[10]),
                                    activated<GATED, OutT>(scaled(gs.w, sx, sw[3])) * scaled(us.w, sx, sw[11])};
                store4<OutT>(Y + (int64_t)m * out_n + (n0 >> 1) + 8 * t + 4 * h, v, whole, 4);
            }
        }
    }
    __syncwarp();
    if (ranks > 1) cluster_sync();                                            // nobody leaves while its tile is being read
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------
// Prompts: persistent pairs of SMs (cta_group::2), W as the 256-row operand, `tile` tokens (a multiple of 32 up to 256) as the other one.  Each block of a
// pair loads its own 128 rows of W and half of the tokens, the instruction reads both blocks' shared memory, and each block's tensor
// memory receives the accumulator of its own rows of W, twice (a tile's drain runs under the next one's products).
//   full[s]       in the leader (rank 0): both blocks' copies report their bytes there
//   empty[s]      in each block: the leader's commit arrives at both
//   acc_full[b]   in each block: likewise, when a tile's accumulator is complete
//   acc_empty[b]  in the leader: the drain warps of both blocks arrive there
constexpr int DRAIN_SETS = 4, DRAIN_WARPS = 4 * DRAIN_SETS, PAIR_THREADS = 64 + 32 * DRAIN_WARPS;
constexpr int PAIR_STAGES = 6;

// The order of the tiles: bands of at most 16 tiles of tokens, all tiles of W inside a band, the tokens fastest, so that a band's tokens stay in the L2
// while W passes.
constexpr int BAND_TILES = 16;
__device__ __forceinline__ void tile_place(int tile, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int bands = (tiles_m + BAND_TILES - 1) / BAND_TILES, high = (tiles_m + bands - 1) / bands;
    const int band = tile / (high * tiles_n), inside = tile - band * high * tiles_n;
    const int own = min(high, tiles_m - band * high);        // the last band may be lower
    tn = inside / own;
    tm = band * high + inside - tn * own;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// 16 lanes by 32 columns of tensor memory as the products' accumulators lie in registers: r[4 j], r[4 j + 1] of lane l are row l / 4, columns
// 8 j + 2 (l % 4) and the next, r[4 j + 2], r[4 j + 3] the same columns eight rows further.
__device__ __forceinline__ void tc_ld_16x32(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}

// What a warp of the drain does with 32 tokens (`live` of them there are, from `m` on, with scales `sx`) of its 32 rows of W at `row0`: columns of tensor
// memory from `acc` on.  `words`: rows of Y are whole 4-byte words.
//
// Without a gate a lane reads its own row.  bfloat16: two tokens make a word; lanes next to each other exchange, and one takes both rows for the
// even token, the other for the odd one: 64 consecutive bytes a token and instruction.
template <typename OutT>
__device__ __forceinline__ void drain_plain(uint32_t acc, const float* sx, float sw, OutT* Y, int64_t m, int live, int row0, int lane, int N, bool words) {
    uint32_t r[32];
    tc_ld32(acc, r);
    tc_wait_ld();
    float v[32];
#pragma unroll
    for (int t = 0; t < 32; t += 4) {
        const float4 x4 = *reinterpret_cast<const float4*>(sx + t);
        v[t] = scaled((int)r[t], x4.x, sw);
        v[t + 1] = scaled((int)r[t + 1], x4.y, sw);
        v[t + 2] = scaled((int)r[t + 2], x4.z, sw);
        v[t + 3] = scaled((int)r[t + 3], x4.w, sw);
    }
    const int row = row0 + lane;
    if (sizeof(OutT) == 4 || !words) {
        if (row >= N) return;
        OutT* to = Y + m * N + row;
#pragma unroll
        for (int t = 0; t < 32; ++t, to += N)
            if (t < live) *to = to_out<OutT>(v[t]);
    } else {
        const int odd = lane & 1;
        const uint32_t both = odd ? 0x3276u : 0x5410u;       // halves of the lane's word and the other's, the even row first
        const int there = row < N ? live - odd : 0;
        OutT* to = Y + (m + odd) * N + (row & ~1);
#pragma unroll
        for (int t = 0; t < 32; t += 2, to += 2 * (int64_t)N) {
            const uint32_t own = pack_bf16(v[t], v[t + 1]), other = __shfl_xor_sync(0xffffffffu, own, 1);
            if (t < there) *reinterpret_cast<uint32_t*>(to) = __byte_perm(own, other, both);
        }
    }
}
// With a gate the rows are gate[8] up[8] gate[8] up[8] of 16 features, and a lane reads a gate's row and its up's, of two tokens in eight.
template <int GATED, typename OutT>
__device__ __forceinline__ void drain_gated(uint32_t acc, const float* sx, const float (&sw)[4], OutT* Y, int64_t m, int live, int row0, int lane, int N,
                                            bool words) {
    const int64_t out_n = N >> 1;
    const int quad = lane >> 2, odd = quad & 1, first = 2 * (lane & 3);
    const uint32_t both = odd ? 0x3276u : 0x5410u;
    uint32_t r[2][16];
    tc_ld_16x32(acc, r[0]);
    tc_ld_16x32(acc + (16u << 16), r[1]);
    tc_wait_ld();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bool whole = row0 + 16 * h + 16 <= N;
        const int feature = (row0 >> 1) + 8 * h + quad;
        OutT* to = Y + (m + first) * out_n + feature;
#pragma unroll
        for (int j = 0; j < 4; ++j, to += 8 * out_n) {
            const float2 s = *reinterpret_cast<const float2*>(sx + 8 * j + first);
            const float y0 = activated<GATED, OutT>(scaled((int)r[h][4 * j], s.x, sw[2 * h])) * scaled((int)r[h][4 * j + 2], s.x, sw[2 * h + 1]);
            const float y1 = activated<GATED, OutT>(scaled((int)r[h][4 * j + 1], s.y, sw[2 * h])) * scaled((int)r[h][4 * j + 3], s.y, sw[2 * h + 1]);
            const int token = 8 * j + first;
            if (sizeof(OutT) == 4 || !words) {
                if (whole && token < live) to[0] = to_out<OutT>(y0);
                if (whole && token + 1 < live) to[out_n] = to_out<OutT>(y1);
            } else {
                const uint32_t own = pack_bf16(y0, y1), other = __shfl_xor_sync(0xffffffffu, own, 4);
                if (whole && token + odd < live) *reinterpret_cast<uint32_t*>(odd ? to + out_n - 1 : to) = __byte_perm(own, other, both);
            }
        }
    }
}

template <int GATED, typename OutT>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Product p, int tile, int* __restrict__ status) {
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(16) float token_scales[DRAIN_WARPS][256 / DRAIN_SETS];       // of a drain warp's share of the tile
    constexpr int STAGES = PAIR_STAGES, BN = 2 * BM;
    constexpr int X_BYTES = BM * BK, W_BYTES = BM * BK, STAGE_BYTES = X_BYTES + W_BYTES;
    constexpr uint32_t TMEM_COLS = 512;                       // two accumulators of 256 columns
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = base + STAGES * STAGE_BYTES;       // full[S], empty[S], acc_full[2], acc_empty[2], slot
    const uint32_t bar_acc_full = bars + 2 * STAGES * 8, bar_acc_empty = bar_acc_full + 16, tmem_slot = bar_acc_empty + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int tiles_m = (p.M + tile - 1) / tile, tiles_n = (p.N + BN - 1) / BN, tiles = tiles_m * tiles_n;
    const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;
    const int nkb = (p.K + BK - 1) / BK;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bars + s * 8, 1);
            mbar_init(bars + (STAGES + s) * 8, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar_acc_full + b * 8, 1);
            mbar_init(bar_acc_empty + b * 8, 2 * DRAIN_WARPS);     // one arrival per drain warp of the pair
        }
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                           // the peer's barriers exist before anything signals them
    tc_fence_after();
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");

    if (warp == 0) {
        pdl_wait();                                           // X is the output of the kernel before
        uint32_t it = 0;
        bool ok = true;
        for (int i = first; i < tiles && ok; i += stride) {
            int tm, tn;
            tile_place(i, tiles_m, tiles_n, tm, tn);
            const int m0 = tm * tile + (int)rank * (tile / 2), n0 = tn * BN + (int)rank * BM;
            for (int kb = 0; kb < nkb; ++kb, ++it) {
                const uint32_t s = it % STAGES;
                ok = mbar_wait_warp(bars + (STAGES + s) * 8, ((it / STAGES) & 1u) ^ 1u);
                if (!ok) {
                    if (lane == 0) atomicExch(status, 1);
                    break;
                }
                const uint32_t x = base + s * STAGE_BYTES, w = x + X_BYTES;
                const uint32_t full_in_leader = map_to_rank(bars + s * 8, 0);
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(bars + s * 8, 2 * (tile / 2 * BK + W_BYTES));       // both blocks' bytes
                    tma_load_2d_pair(x, &map_x, full_in_leader, kb * BK, m0);
                    tma_load_2d_pair(w, &map_w, full_in_leader, kb * BK, n0);
                }
                __syncwarp();
            }
        }
        wait_for_stages<STAGES>(bars + STAGES * 8, it);
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = make_idesc_i8(2 * BM, tile);
            const uint64_t desc0 = desc_k_major(base);
            uint32_t it = 0, local = 0;
            bool ok = true;
            tmem_base = __shfl_sync(0xffffffffu, tmem_base, 0);
            for (int i = first; i < tiles && ok; i += stride, ++local) {
                const uint32_t buf = local & 1u;
                ok = mbar_wait_warp(bar_acc_empty + buf * 8, ((local >> 1) & 1u) ^ 1u);      // both blocks have drained it
                if (!ok) {
                    if (lane == 0) atomicExch(status, 4);
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem_base + buf * 256u;
                for (int kb = 0; kb < nkb; ++kb, ++it) {
                    const uint32_t s = it % STAGES;
                    ok = mbar_wait_warp(bars + s * 8, (it / STAGES) & 1u);
                    if (!ok) {
                        if (lane == 0) atomicExch(status, 2);
                        break;
                    }
                    tc_fence_after();
                    const uint64_t dx = desc0 + (uint64_t)(s * (STAGE_BYTES >> 4)), dw = dx + (X_BYTES >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k)
                            tc_mma_pair_i8(acc, dw + (uint64_t)(k * 2), dx + (uint64_t)(k * 2), idesc, (kb > 0 || k > 0) ? 1u : 0u);
                        tc_commit_pair(bars + (STAGES + s) * 8);
                    }
                    __syncwarp();
                }
                if (elect_one()) tc_commit_pair(bar_acc_full + buf * 8);
                __syncwarp();
            }
        }
    } else {
        pdl_wait();
        // 32 rows of W by a share of the tile's tokens
        const int lane_base = (warp & 3) * 32, set = (warp - 2) >> 2, share = tile / DRAIN_SETS, c0 = set * share;
        OutT* Y = (OutT*)p.y;
        const bool words = (reinterpret_cast<uintptr_t>(Y) & 3u) == 0 && p.N % 2 == 0;      // (with a gate N / 2 is even, too)
        float* sx = token_scales[warp - 2];
        uint32_t local = 0;
        for (int i = first; i < tiles; i += stride, ++local) {
            const uint32_t buf = local & 1u;
            int tm, tn;
            tile_place(i, tiles_m, tiles_n, tm, tn);
            const int m0 = tm * tile + c0, row0 = tn * BN + (int)rank * BM + lane_base;
            const int tokens = min(share, p.M - m0);         // none or less where the share lies behind the last token
            __syncwarp();
            for (int t = lane; t < share; t += 32) sx[t] = t < tokens ? p.sx[m0 + t] : 0.0f;
            float sw[4];                                     // of the rows that the lane reads
#pragma unroll
            for (int i = 0; i < (GATED ? 4 : 1); ++i) {
                const int row = row0 + (GATED ? 8 * i + (lane >> 2) : lane);
                sw[i] = row < p.N ? p.sw[row] : 0.0f;
            }
            __syncwarp();
            if (!mbar_wait(bar_acc_full + buf * 8, (local >> 1) & 1u)) {
                if (lane == 0) atomicExch(status, 3);
                break;
            }
            __syncwarp();
            tc_fence_after();
            const uint32_t acc = tmem_base + ((uint32_t)lane_base << 16) + buf * 256u + (uint32_t)c0;
#pragma unroll 1
            for (int c = 0; c < tokens; c += 32) {
                if constexpr (GATED != 0) drain_gated<GATED, OutT>(acc + (uint32_t)c, sx + c, sw, Y, m0 + c, tokens - c, row0, lane, p.N, words);
                else drain_plain<OutT>(acc + (uint32_t)c, sx + c, sw[0], Y, m0 + c, tokens - c, row0, lane, p.N, words);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_rank(bar_acc_empty + buf * 8, 0));
        }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync();                                           // the peer reads this block's memory and barriers until here
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// Tokens of a tile, stages and blocks an SM: more blocks with shorter rings where two an SM do not hold all.
#define Q3_BY_TILE(M, N, SPLITS, CALL)                                                            \
    do {                                                                                          \
        const bool more = (int64_t)(((N) + BM - 1) / BM) * (SPLITS) > 2 * q3_device_sm_count();   \
        if ((M) <= 16) { if (more) CALL(16, 4, 3); CALL(16, 5, 2); }                              \
        if ((M) <= 32) { if (more) CALL(32, 3, 3); CALL(32, 5, 2); }                              \
        if ((M) <= 64) { if (more) CALL(64, 3, 3); CALL(64, 4, 2); }                              \
        if ((M) <= 128) { if (more) CALL(128, 2, 3); CALL(128, 3, 2); }                           \
        CALL(256, 4, 1);                                                                          \
    } while (0)

constexpr int mid_shared(int tile, int stages) {
    const int ring = stages * (BM * BK + tile * BK), part = (tile * PART_LD * 4 + 1023) / 1024 * 1024;
    return (ring > part ? ring : part) + 1024 + 256;
}

template <int MT, int STAGES, int MINB, int GATED, typename OutT> int launch_mid(const Product& p, int splits, int* status, cudaStream_t stream) {
    constexpr int SMEM = mid_shared(MT, STAGES);
    static Q3PerDevice configured;
    const cudaError_t e = q3_allow_shared_memory(mid_kernel<MT, STAGES, MINB, GATED, OutT>, SMEM, configured);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_w, map_x;
    if (!q3_make_map_bytes(&map_w, p.w, p.N, p.K, p.ldw, BM) || !q3_make_map_bytes(&map_x, p.x, p.M, p.K, p.ldx, MT)) return Q3_ERR_BAD_SIZE;
    const int64_t token_tiles = (p.M + MT - 1) / MT;
    if (token_tiles > GRID_YZ) return Q3_ERR_TOO_LARGE;
    return (int)q3_launch_cluster(mid_kernel<MT, STAGES, MINB, GATED, OutT>, dim3((p.N + BM - 1) / BM, splits, (unsigned)token_tiles), dim3(THREADS),
                                  (size_t)SMEM, stream, dim3(1, splits, 1), map_w, map_x, p, status);
}

// ---------------------------------------------------------------------------------------------
// Which form takes a product, in how many K ranges or tokens a tile: the one whose estimate is least.  Microseconds of a launch among others, W from
// memory, but for a constant that all have.  The other constants are fitted so that what they choose of 7,900 times of 1,000 products (1 to 8,000 tokens, 64
// to 25,600 channels and widths, plain and gated) is near the best of each product: 1.9 % slower in the mean, 7 % or more for one in ten (2.1 and 8 %
// for 700 other products; 150 drawn later, on another device, 2.6 and 10 %, the worst 37 %).
inline int cuts(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Steps of 64 a warp, as many blocks as run at once (see `few`); where a wave is not full what a step costs is latency.
float few_us(int M, int N, int K) {
    const int sms = q3_device_sm_count(), rows = cuts(N, 16), tiles = M <= 8 ? 1 : M <= 16 ? 2 : 4;
    const bool once = rows <= 2 * sms;
    const int warps = tiles < 4 && once ? 16 : 8, slots = tiles == 4 || once ? 2 : tiles == 2 || (rows <= 3 * sms && K >= 8192) ? 3 : 4;
    const float waves = (float)((int64_t)rows * cuts(M, 8 * tiles)) / (float)(slots * sms);
    const float step = 0.273f + fminf(waves, 1.0f) * (float)(warps * slots) / 32.0f * (tiles == 1 ? 0.146f : tiles == 2 ? 0.47f : 0.82f);
    return -0.53f + fmaxf(waves, 1.0f) * (0.35f * (float)tiles + (float)cuts(cuts(K, 64), warps) * step);
}
// Steps of 128 a block: latency, or the bytes of the blocks that share an SM.  Then the tile's way through shared memory and out.  Not all places are
// taken by clusters: the SMs come in groups, and a group whose places are no multiple of a cluster leaves some empty.
float mid_us(int M, int N, int K, int splits) {
    const int sms = q3_device_sm_count(), tile = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : M <= 128 ? 128 : 256, rows = cuts(N, BM);
    const int tokens = cuts(M, tile);
    if (tokens > GRID_YZ) return 1e30f;                        // more tiles of tokens than a grid takes
    const int an_sm = tile == 256 ? 1 : (int64_t)rows * splits > 2 * sms ? 3 : 2;
    const float taken = splits <= 2 ? 1.0f : tile == 256 ? (splits == 3 ? 0.91f : splits <= 6 ? 0.89f : 0.81f) : splits <= 4 ? 0.96f : 0.89f;
    const int64_t blocks = (int64_t)rows * splits * tokens;
    const int slots = most((int)((float)(an_sm * sms) * taken), 1), waves = cuts(blocks, slots);
    const float shared = (float)(waves == 1 ? (int)blocks : slots) / (float)sms, t = (float)tile / 64.0f;
    const float step = fmaxf(0.214f + 0.03f * t, shared * (16.0f + 8.0f * t) * 0.0085f);
    const float around = 1.34f * t + 1.21f * shared + (splits > 1 ? 0.08f : 0.0f);
    return 0.24f + fmaxf((float)waves * ((float)cuts(cuts(K, BK), splits) * step + around), (float)N * (float)K * (float)tokens / 14e6f);
}
// Steps of 128 a pair: the products, the copies of few tokens, or what the L2 gives all pairs; a tile's drain under the next one's steps, but for the last.
float pair_us(int M, int N, int K, int tile) {
    const int pairs = most(q3_device_sm_count() / 2, 1);
    const int64_t tiles = (int64_t)cuts(M, tile) * cuts(N, 256);
    const float t = (float)tile / 256.0f, full = fminf((float)tiles / (float)pairs, 1.0f);
    const float step = fmaxf(fmaxf(0.1835f, 0.335f * t), 0.1525f * full * (t + 1.0f)), drain = 1.23f + 0.77f * t;
    return 0.03f * t + (float)cuts(tiles, pairs) * fmaxf((float)cuts(K, BK) * step, drain) + drain;
}

struct Choice {
    int splits;
    float us;
};
Choice mid_choice(int M, int N, int K) {
    Choice best{1, mid_us(M, N, K, 1)};
    for (int s : {2, 3, 4, 6, 8}) {
        const float us = s <= cuts(K, BK) ? mid_us(M, N, K, s) : best.us;
        if (us < best.us) best = Choice{s, us};
    }
    return best;
}
// Equal tiles of a multiple of 32 tokens: those that whole 256s, or one to three more, would make, and smaller ones where these fill the pairs.
Choice pair_choice(int M, int N, int K) {
    Choice best{256, 1e30f};
    auto take = [&](int tile) {
        const float us = pair_us(M, N, K, tile);
        if (us < best.us) best = Choice{tile, us};
    };
    for (int n = cuts(M, 256); n < cuts(M, 256) + 4; ++n) take(cuts(cuts(M, n), 32) * 32);
    for (int tile = 32; tile < 160 && tile - 32 < M; tile += 32) take(tile);
    return best;
}

template <int GATED, typename OutT> int mid(const Product& p, int splits, int* status, cudaStream_t stream) {
    const int nkb = (p.K + BK - 1) / BK;
    if (splits == 0) splits = mid_choice(p.M, p.N, p.K).splits;
    if (splits > nkb) splits = nkb;
#define Q3_MID(MT, ST, MB) return launch_mid<MT, ST, MB, GATED, OutT>(p, splits, status, stream)
    Q3_BY_TILE(p.M, p.N, splits, Q3_MID);
#undef Q3_MID
}

template <int GATED, typename OutT> int pair(const Product& p, int tile, int* status, cudaStream_t stream) {
    constexpr int SMEM = PAIR_STAGES * (2 * BM * BK) + 1024 + 256;
    const auto kernel = pair_kernel<GATED, OutT>;
    static Q3PerDevice configured;
    const cudaError_t e = q3_allow_shared_memory(kernel, SMEM, configured);
    if (e != cudaSuccess) return (int)e;
    if (tile == 0) tile = pair_choice(p.M, p.N, p.K).splits;
    if (tile < 32 || tile > 256 || tile % 32 != 0) return Q3_ERR_BAD_SIZE;
    CUtensorMap map_x, map_w;
    if (!q3_make_map_bytes(&map_x, p.x, p.M, p.K, p.ldx, tile / 2) || !q3_make_map_bytes(&map_w, p.w, p.N, p.K, p.ldw, BM)) return Q3_ERR_BAD_SIZE;
    const int64_t tiles = (int64_t)((p.M + tile - 1) / tile) * ((p.N + 255) / 256);
    if (tiles > 0x3fffffff) return Q3_ERR_TOO_LARGE;
    const int most_pairs = most(q3_device_sm_count() / 2, 1), pairs = tiles < most_pairs ? (int)tiles : most_pairs;
    return (int)q3_launch_cluster(kernel, dim3(2 * pairs), dim3(PAIR_THREADS), (size_t)SMEM, stream, dim3(2, 1, 1), map_x, map_w, p, tile, status);
}

// The kernels' 32-bit row numbers run on to the end of a tile of at most 256.
constexpr int MOST_ROWS = 0x7fffffff - 256;
int product_of(const q3_gemm_int8_args& a, Product& p) {
    if (a.rows > MOST_ROWS || a.channels > MOST_ROWS) return Q3_ERR_TOO_LARGE;
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

// Few tokens, W streamed (any number is taken; W is read once for every 8, 16 or 32 of them).
Q3_EXPORT int q3_gemm_int8_few(const q3_gemm_int8_args* a) {
    if (a->rows <= 0 || a->channels <= 0) return 0;
    Product p;
    const int bad = product_of(*a, p);
    if (bad) return bad;
#define Q3_FEW(G, T) few<G, T>(p, (cudaStream_t)a->stream)
    Q3_BY_EPILOGUE(Q3_FEW);
#undef Q3_FEW
}

// Up to some hundred tokens: weights first on tcgen05, `splits` K ranges in a cluster (0: chosen).
Q3_EXPORT int q3_gemm_int8_mid(const q3_gemm_int8_args* a) {
    if (a->rows <= 0 || a->channels <= 0) return 0;
    Product p;
    const int bad = product_of(*a, p);
    if (bad) return bad;
    if (a->splits < 0 || a->splits > 8) return Q3_ERR_BAD_SIZE;
#define Q3_MIDDLE(G, T) mid<G, T>(p, a->splits, (int*)a->status, (cudaStream_t)a->stream)
    Q3_BY_EPILOGUE(Q3_MIDDLE);
#undef Q3_MIDDLE
}

// Prompts: pairs of SMs, tiles of `splits` tokens (a multiple of 32 up to 256; 0: chosen) by 256 rows of W.
Q3_EXPORT int q3_gemm_int8_pair(const q3_gemm_int8_args* a) {
    if (a->rows <= 0 || a->channels <= 0) return 0;
    Product p;
    const int bad = product_of(*a, p);
    if (bad) return bad;
#define Q3_PAIR(G, T) pair<G, T>(p, a->splits, (int*)a->status, (cudaStream_t)a->stream)
    Q3_BY_EPILOGUE(Q3_PAIR);
#undef Q3_PAIR
}

// The form that a product of these sizes should go to, and the `splits` of it: 0 few tokens, 1 weights first, 2 pairs of SMs.
Q3_EXPORT int q3_gemm_int8_plan(int rows, int channels, int width, int* splits) {
    *splits = 0;
    if (rows <= 0 || channels <= 0 || width <= 0) return 0;
    const Choice m = mid_choice(rows, channels, width), p = pair_choice(rows, channels, width);
    if (rows <= 64 && few_us(rows, channels, width) <= fminf(m.us, p.us)) return 0;
    *splits = m.us <= p.us ? m.splits : p.splits;
    return m.us <= p.us ? 1 : 2;
}
