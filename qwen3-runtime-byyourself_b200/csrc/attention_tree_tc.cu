// Attention of a step's new tokens over the cache's pages in bfloat16 or in 8 bits on the 5th-generation tensor cores, for trees (or runs) whose
// rows - a row is a token and a query head - fill tiles of 128.  What a token sees and what comes out is said in attention_tree.cu.
//
// S = Q K^T and O += P V are tcgen05.mma of 128 rows and 128 keys with their accumulators in tensor memory.  A block (one an SM) takes two
// tiles of 128 rows of one kv head at a time, so that a stretch of 128 keys is brought in once for both and the products of one tile run
// under the softmax of the other; the stretches of all items are shared out evenly over the blocks (tree_work.cuh).
//   warps 0-7    softmax: thread r of a tile's 128 owns row r (TMEM lane r).  It reads its scores twice, for the maximum and for the
//                weights, 32 at a time, so that 120 registers do; writes the weights over the scores, and rescales O when the maximum is raised by
//                more than 2^8.  At the end of a part it writes the row, or its share of it for the second kernel to add up.
//   warps 8-11   bring in the keys, warps 12-15 the values.  bfloat16: by TMA; 8 bits: a warp loads codes a stretch ahead into registers, turns
//                them into half precision, which holds them exactly, and stores them where TMA would have put them.
//   warp 16      issues the products, one elected thread.  (Warps 17-19 make its group of four whole, which registers are handed out to.)
//
// 8 bits.  A stretch's keys are brought to one scale, that of its first row, 2^k0, by folding 2^(k - k0) into the half-precision numbers, which is exact
// for k - k0 in -15 .. 7; so are its values.  Scores are then multiplied by 2^k0 with the softmax's own scale; v0 is added to the scores in log2 units, so
// that a weight is w = 2^(x + v0 - M) with M the running maximum of x + v0 and the sum of the softmax that of w 2^-v0.  Where some row of a stretch has a scale outside that
// range, what is missing (`rest`) is added score by score, in a path of its own.  Queries are brought into half precision as in attention_tree_mma.cu.
//
// A value that is no number (infinity, NaN) in a stretch that some row does not see in whole is taken out before the product, and put into the
// outputs of the rows that see it: 0 times a NaN would reach the others.
// What bounds it: a stretch of 128 keys and 256 rows is 2,048 cycles of the tensor pipe and as many of the special-function unit (an exponential a score).
// Every mbarrier wait is bounded and reports into `status`.
#include <cuda.h>

#include "page8.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"
#include "tree_work.cuh"

#ifndef Q3_HEAD_DIM
#error "compile with -DQ3_HEAD_DIM=<64 or 128>"
#endif

namespace {

constexpr int D = Q3_HEAD_DIM, PAGE = Q3_PAGE_TOKENS;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
static_assert(PAGE == 64, "a stretch is two pages of 64 keys");
constexpr int BM = 128, ROWS = 2 * BM, STRETCH = 2 * PAGE, HALVES = D / 64;
constexpr int SOFTMAX_WARPS = 8, BRING_WARPS = 4, V_WARP = 12, MMA_WARP = 16, THREADS = 20 * 32;
// Registers of a thread by role: 256 x 144 + 256 x 80 + 128 x 32 = 640 x 96, what the block is launched with.
constexpr int LAUNCH_REGS = 96, SOFTMAX_REGS = 144, BRING_REGS = 80, MMA_REGS = 32;
static_assert(8 * 32 * SOFTMAX_REGS + 8 * 32 * BRING_REGS + 4 * 32 * MMA_REGS <= THREADS * LAUNCH_REGS, "shares of the launch's registers");
constexpr int STAGES = 2, NOTES = 4;                      // stretches of keys and of values in shared memory; what is noted of a stretch lives longer
constexpr int HALF_BYTES = BM * 128, TILE_BYTES = HALVES * HALF_BYTES;                     // 128 rows of 128 bytes; a tile of queries, keys or values
constexpr int PANEL_BYTES = PAGE * 128;                   // a page's 64 rows of 128 bytes
constexpr uint32_t TMEM_COLS = 512, COL_S = 0, COL_O = 256;   // S (and P over it) of tile x at x * 128, O at 256 + x * 128
constexpr float RAISE = 8.0f;
constexpr int FOLD_LOW = -15, FOLD_HIGH = 7;
constexpr int PART = ROWS * (D + 2);                      // float32 of a part: sums [D / 4][ROWS][4], then (maximum, sum) [ROWS][2]

struct Note {                                             // what is noted of a stretch in 8 bits
    float scale;                                          // 2^k0 (values: v0)
    uint32_t flags[BRING_WARPS];                          // bit 0: some scale is out of range; bit 1: some value is no number
    uint32_t pad[3];
};
struct Shared {
    Note keys[NOTES], values[NOTES];
    float key_rest[NOTES][STRETCH], value_rest[NOTES][STRETCH];
    TreeShare share;
    unsigned long long bars[1 + 5 * STAGES + 6 + NOTES];
    uint32_t tmem;
};
constexpr int SMEM_BYTES = 2 * TILE_BYTES + 2 * STAGES * TILE_BYTES + (int)sizeof(Shared);
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of a block");

struct Args {
    TreeStep step;
    const bf16* q;
    bf16* out;
    const unsigned char *keys, *values;
    const uint8_t *key_scales, *value_scales;
    float* parts;
    int* status;
    float scale_log2;
};

using Work = TreeWork<STRETCH, ROWS>;

__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// kind::f16 instruction descriptor: float32 accumulator, operands both half precision or both bfloat16; bit 16 = B is MN-major.
constexpr uint32_t idesc(bool half, int m, int n, bool b_mn_major) {
    return (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <bool HALF> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (HALF) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
// The values of a word that are infinities or NaNs, each marked by all of its bits.
template <bool F8> __device__ __forceinline__ uint32_t no_numbers(uint32_t w) {
    if constexpr (F8) return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
    else return ((((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// 16-byte chunk `c` (of D / 8) of row r of a tile whose halves of 64 columns are `half_bytes` apart, as TMA's 128-byte swizzle lays it.
__device__ __forceinline__ uint32_t chunk_at(int r, int c, int half_bytes) { return (uint32_t)((c >> 3) * half_bytes + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// A page number of a sequence, within the cache whatever the table says.
__device__ __forceinline__ int64_t page_of(const TreeStep& st, const int* table, int i) {
    const int p = i < st.pages_per_seq ? table[i] : 0;
    return p >= 0 && p < st.n_pages ? p : 0;
}

// Where the values of an output row are that are no numbers: bit d of `plus` for +infinity, of `minus` for -infinity, of both for NaN.
struct Odd {
    uint32_t plus[D / 32], minus[D / 32];
    bool any;
};

// The values of stretch `s` that are no numbers, of the keys that the row sees (bits lo: the first 64, hi: the others).
template <bool F8>
__device__ __noinline__ void find_odd(const Args& a, const int* table, int head, int s, unsigned long long lo, unsigned long long hi, Odd& odd) {
    for (int key = 0; key < STRETCH; ++key) {
        if (!((key < 64 ? lo >> key : hi >> (key - 64)) & 1)) continue;
        const int64_t cell = (page_of(a.step, table, 2 * s + (key >> 6)) * a.step.nkv + head) * PAGE + (key & 63);
        constexpr int WORDS = D * (F8 ? 1 : 2) / 4, EACH = F8 ? 4 : 2, BITS = F8 ? 8 : 16;
        const uint32_t* row = reinterpret_cast<const uint32_t*>(a.values + cell * (D * (F8 ? 1 : 2)));
        for (int w = 0; w < WORDS; ++w) {
            const uint32_t v = row[w], bad = no_numbers<F8>(v);
            if (bad == 0) continue;
            odd.any = true;
            for (int e = 0; e < EACH; ++e) {
                if (!(bad >> (BITS * e) & 1u)) continue;
                const uint32_t x = v >> (BITS * e) & (F8 ? 0xffu : 0xffffu);
                const bool infinite = !F8 && (x & 0x7fu) == 0u;
                const int d = w * EACH + e;
                if (!infinite || !(x >> 15)) odd.plus[d >> 5] |= 1u << (d & 31);
                if (!infinite || (x >> 15)) odd.minus[d >> 5] |= 1u << (d & 31);
            }
        }
    }
}

template <bool F8>
__global__ void __launch_bounds__(THREADS, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Args a) {
    extern __shared__ unsigned char smem[];
    pdl_launch_dependents();
    const uint32_t base = smem_u32(smem);
    const uint32_t q_smem = base, k_smem = base + 2 * TILE_BYTES, v_smem = k_smem + STAGES * TILE_BYTES;
    Shared& sh = *reinterpret_cast<Shared*>(smem + 2 * TILE_BYTES + 2 * STAGES * TILE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bars = smem_u32(sh.bars);
    const uint32_t bar_q = bars, bar_k_full = bars + 8, bar_k_empty = bar_k_full + 8 * STAGES, bar_v_full = bar_k_empty + 8 * STAGES;
    const uint32_t bar_v_empty = bar_v_full + 8 * STAGES, bar_v_here = bar_v_empty + 8 * STAGES;      // v_here: TMA's values, before they are looked through
    const uint32_t bar_s_full = bar_v_here + 8 * STAGES, bar_p_full = bar_s_full + 16, bar_pv_done = bar_p_full + 16;   // one a tile
    const uint32_t bar_noted = bar_pv_done + 16;         // what is noted of a stretch's keys can be read
    if (base & 1023u) {                                  // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) atomicExch(a.status, 40);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(bar_q, SOFTMAX_WARPS);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_k_full + 8 * s, F8 ? BRING_WARPS : 1);
            mbar_init(bar_k_empty + 8 * s, 1);
            mbar_init(bar_v_full + 8 * s, BRING_WARPS);
            mbar_init(bar_v_empty + 8 * s, 1);
            mbar_init(bar_v_here + 8 * s, 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(bar_s_full + 8 * x, 1);
            mbar_init(bar_p_full + 8 * x, 4);
            mbar_init(bar_pv_done + 8 * x, 1);
        }
        for (int n = 0; n < NOTES; ++n) mbar_init(bar_noted + 8 * n, BRING_WARPS);
        mbar_init_fence();
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    const TreeStep& st = a.step;
    if (warp == 0) {
        const TreeShare found = Work::share(st, 1, blockIdx.x, gridDim.x);
        if (lane == 0) sh.share = found;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    TreeShare share = sh.share;
    const int group = st.nq / st.nkv;
    auto failed = [&](int where) { if (lane == 0) atomicExch(a.status, where); };

    if (warp < SOFTMAX_WARPS) {
        // ------------------------------------------------ softmax: thread = row
        const int x = warp >> 2, r = (warp & 3) * 32 + lane;                         // tile, row of it
        const uint32_t t_row = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_s = t_row + COL_S + x * 128, t_o = t_row + COL_O + x * 128;
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        int stretch = 0;                                                             // of this block, over all parts
        uint32_t turn = 0, q_turn = 0;                                               // of this tile's barriers, of the parts
        bool ok = true;
        for (int at = share.from; at < share.to && ok;) {
            const TreePart part = Work::part(st, share, at, blockIdx.x);
            const int t0 = st.seq_start[part.seq], n_new = Work::n_new(st, part.seq), pos0 = st.seq_pos0[part.seq];
            const int row0 = part.tile * ROWS, rows = n_new * group - row0 - x * BM;      // of this tile
            const int steps = part.end - part.begin;
            const int* table = st.page_table + (int64_t)part.seq * st.pages_per_seq;
            // ---- this row's query
            const int row = row0 + x * BM + r, own = min(row / group, n_new - 1);
            bf16* const out = a.out + ((int64_t)(t0 + own) * st.nq + part.head * group + row % group) * D;
            float factor = a.scale_log2;
            if (rows > 0) {
                const uint4* src = reinterpret_cast<const uint4*>(a.q + ((int64_t)(t0 + own) * st.nq + part.head * group + row % group) * D);
                const uint32_t dst = q_smem + x * TILE_BYTES;
                float down = 1.0f;
                if constexpr (F8) {
                    uint32_t top = 0;
                    for (int c = 0; c < D / 8; ++c) {
                        const uint4 w = src[c];
                        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = max(top, max(v[e] & 0x7fffu, v[e] >> 16 & 0x7fffu));
                    }
                    int e2 = (int)(top >> 7) - 127;
                    e2 = e2 >= 128 ? 0 : min(max(e2, -60), 60);
                    down = q3_exp2i(-e2);
                    factor *= q3_exp2i(e2);
                }
                for (int c = 0; c < D / 8; ++c) {
                    uint4 w = src[c];
                    if constexpr (F8) {
                        uint32_t* v = &w.x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = pack2<true>(__uint_as_float(v[e] << 16) * down, __uint_as_float(v[e] & 0xffff0000u) * down);
                    }
                    if (r >= rows) w = make_uint4(0, 0, 0, 0);
                    st_shared_v4(dst + chunk_at(r, c, HALF_BYTES), w);
                }
                fence_proxy_async();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_q);
            if (rows <= 0) {                                                         // no second tile: on to the next part with the first tile's warps
                ok = mbar_wait_warp(bar_q, q_turn);
                if (!ok) { failed(39); break; }
                q_turn ^= 1u;
                stretch += steps;
                at = Work::next(share, at, part);
                continue;
            }

            q_turn ^= 1u;

            float m_run = -INFINITY, l_run = 0.0f;
            const unsigned long long* mask = st.tree != nullptr ? st.tree + (int64_t)(t0 + own) * st.words : nullptr;
            Odd odd;
            odd.any = false;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) odd.plus[i] = odd.minus[i] = 0u;
            for (int i = 0; i < steps; ++i, ++stretch) {
                const int key0 = (part.begin + i) * STRETCH, note = stretch % NOTES;
                const bool edge = key0 + STRETCH > pos0;                             // some key is a new token's, or behind the end
                ok = mbar_wait_warp(bar_s_full + 8 * x, turn & 1u);
                if (!ok) { failed(41); break; }
                if (F8 || edge) {                                                    // what is noted of the stretch
                    ok = mbar_wait_warp(bar_v_full + 8 * (stretch % STAGES), (uint32_t)(stretch / STAGES) & 1u) &&
                         (!F8 || mbar_wait_warp(bar_noted + 8 * note, (uint32_t)(stretch / NOTES) & 1u));
                    if (!ok) { failed(42); break; }
                }
                tc_fence_after();
                // ---- of the stretch: score = dot * c1, in log2 units, and v0
                float c1 = factor, v0 = 0.0f;
                bool rests = false;
                if constexpr (F8) {
                    c1 = fmaxf(c1 * sh.keys[note].scale, 1.2e-38f);                  // (what is not seen stays minus infinity)
                    v0 = sh.values[note].scale;
                    uint32_t flags = 0;
#pragma unroll
                    for (int w = 0; w < BRING_WARPS; ++w) flags |= sh.keys[note].flags[w] | sh.values[note].flags[w];
                    rests = flags & 1u;
                }
                uint32_t seen[4] = {~0u, ~0u, ~0u, ~0u};
                if (edge) {
                    const unsigned long long lo = tree_seen(mask, st.words, pos0, n_new, own, key0), hi = tree_seen(mask, st.words, pos0, n_new, own, key0 + 64);
                    seen[0] = (uint32_t)lo;
                    seen[1] = (uint32_t)(lo >> 32);
                    seen[2] = (uint32_t)hi;
                    seen[3] = (uint32_t)(hi >> 32);
                    uint32_t flags = 0;
#pragma unroll
                    for (int w = 0; w < BRING_WARPS; ++w) flags |= sh.values[note].flags[w];
                    if (flags & 2u) find_odd<F8>(a, table, part.head, part.begin + i, lo, hi, odd);
                }
                __syncwarp();
                // ---- the maximum of x + v0 (and the rests)
                float top = -INFINITY;
                uint32_t s[2][32];
                auto scores = [&](int c, uint32_t* v) {                              // 32 scores, those that are not seen minus infinity
                    if (edge) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(seen[c] >> e & 1u)) v[e] = 0xff800000u;
                    }
                };
                tc_ld32(t_s, s[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tc_wait_ld();
                    if (c < 3) tc_ld32(t_s + 32 * (c + 1), s[(c + 1) & 1]);
                    uint32_t* v = s[c & 1];
                    scores(c, v);
                    if (F8 && rests) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            top = fmaxf(top, fmaf(__uint_as_float(v[e]) * sh.key_rest[note][32 * c + e], c1, sh.value_rest[note][32 * c + e]));
                    } else {
                        float mx[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 4]));
#pragma unroll
                        for (int e = 8; e < 32; e += 8)
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(v[e + k]), __uint_as_float(v[e + k + 4]));
                        const float most = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                        top = fmaxf(top, most * c1);
                    }
                }
                top += v0;
                const bool raise = top > m_run + RAISE;
                float alpha = 1.0f;
                if (raise) {
                    alpha = ex2(m_run - top);
                    m_run = top;
                    l_run *= alpha;
                }
                __syncwarp();
                if (i > 0 && __any_sync(0xffffffffu, raise)) {
                    // (the products of the stretch before are done: this stretch's scores were asked for after them)
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        tc_ld32(t_o + c, s[0]);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[0][e] = __float_as_uint(__uint_as_float(s[0][e]) * alpha);
                        tc_st32(t_o + c, s[0]);
                    }
                }
                // ---- weights, over the scores
                const float shift = v0 - (m_run == -INFINITY ? 0.0f : m_run);
                const float2 c2 = make_float2(c1, c1), shift2 = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                tc_ld32(t_s, s[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tc_wait_ld();
                    if (c < 3) tc_ld32(t_s + 32 * (c + 1), s[(c + 1) & 1]);
                    uint32_t* v = s[c & 1];
                    scores(c, v);
                    uint32_t p[16];
                    if (F8 && rests) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            // (where nothing is left by the folds, these are the other path's numbers to the bit: a row does not feel the scales of
                            // keys that it does not see)
                            float w[2];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const float rest = sh.value_rest[note][32 * c + e + k];
                                w[k] = ex2(fmaf(__uint_as_float(v[e + k]) * sh.key_rest[note][32 * c + e + k], c1, shift + rest));
                                float& to_sum = k == 0 ? sum[(e >> 1) & 1].x : sum[(e >> 1) & 1].y;
                                to_sum = fmaf(w[k], ex2(-rest), to_sum);
                            }
                            p[e / 2] = pack2<true>(w[0], w[1]);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 t = __ffma2_rn(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), c2, shift2);
                            const float2 w = make_float2(ex2(t.x), ex2(t.y));
                            sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], w);
                            p[e / 2] = pack2<F8>(w.x, w.y);
                        }
                    }
                    tc_st16(t_s + 16 * c, p);
                }
                const float total = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                l_run += F8 ? total * ex2(-v0) : total;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_p_full + 8 * x);
                turn ^= 1u;
            }
            if (!ok) break;
            ok = mbar_wait_warp(bar_pv_done + 8 * x, turn ^ 1u);                      // the part's last products (turn: as many as there were stretches)
            if (!ok) { failed(43); break; }
            tc_fence_after();
            // ---- the row, or its part of it
            const bool whole = part.parts == 1;
            const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
            float* const dst = a.parts + (int64_t)part.slot * PART;
            const int pr = x * BM + r;                                               // the row among the part's
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                __syncwarp();
                tc_ld32(t_o + c, o);
                tc_wait_ld();
                if (odd.any) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        if (odd.plus[c / 32] >> e & 1u) o[e] = __float_as_uint(__uint_as_float(o[e]) + INFINITY);
                        if (odd.minus[c / 32] >> e & 1u) o[e] = __float_as_uint(__uint_as_float(o[e]) - INFINITY);
                    }
                }
                if (r < rows) {
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint4 v;
                            v.x = pack2<false>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                            v.y = pack2<false>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                            v.z = pack2<false>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
                            v.w = pack2<false>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
                            *reinterpret_cast<uint4*>(out + c + e) = v;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4*>(dst + ((c + e) / 4 * ROWS + pr) * 4) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                }
            }
            if (!whole && r < rows) *reinterpret_cast<float2*>(dst + ROWS * D + 2 * pr) = make_float2(m_run, l_run);
            tc_fence_before();
            at = Work::next(share, at, part);
        }
    } else if (warp < MMA_WARP) {
        // ------------------------------------------------ the keys (warps 8-11) and the values (12-15)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BRING_REGS));
        const bool is_v = warp >= V_WARP;
        const int w4 = warp & 3;
        const uint32_t tiles = is_v ? v_smem : k_smem, bar_full = is_v ? bar_v_full : bar_k_full, bar_empty = is_v ? bar_v_empty : bar_k_empty;
        int stretch = 0;
        bool ok = true;
        for (int at = share.from; at < share.to && ok;) {
            const TreePart part = Work::part(st, share, at, blockIdx.x);
            const int n_new = Work::n_new(st, part.seq), pos0 = st.seq_pos0[part.seq], steps = part.end - part.begin;
            const int* table = st.page_table + (int64_t)part.seq * st.pages_per_seq;
            const int key_end = pos0 + n_new;
            if constexpr (F8) {
                // a row is D / 16 lanes' sixteen codes; a warp has 32 rows of a stretch, all of one page
                constexpr int PER_ROW = D / 16, AT_ONCE = 32 / PER_ROW, TURNS = PER_ROW;
                const unsigned char* const source = is_v ? a.values : a.keys;
                const uint8_t* const scale_source = is_v ? a.value_scales : a.key_scales;
                const int c = lane % PER_ROW, r_in = lane / PER_ROW;
                uint4 codes[TURNS];
                uint8_t scale[TURNS], scale0 = 0;
                auto load = [&](int s) {
                    const int64_t first = (page_of(st, table, 2 * s) * st.nkv + part.head) * PAGE;
                    const int64_t cell = (page_of(st, table, 2 * s + (w4 >> 1)) * st.nkv + part.head) * PAGE + (w4 & 1) * 32 + r_in;
                    scale0 = scale_source[first];
#pragma unroll
                    for (int i = 0; i < TURNS; ++i) {
                        codes[i] = *reinterpret_cast<const uint4*>(source + (cell + i * AT_ONCE) * D + c * 16);
                        scale[i] = scale_source[cell + i * AT_ONCE];
                    }
                };
                load(part.begin);
                for (int n = 0; n < steps; ++n, ++stretch) {
                    const int stage = stretch % STAGES, note = stretch % NOTES, key0 = (part.begin + n) * STRETCH;
                    const bool edge = key0 + STRETCH > pos0;
                    ok = mbar_wait_warp(bar_empty + 8 * stage, ((uint32_t)(stretch / STAGES) & 1u) ^ 1u);
                    if (!ok) { failed(is_v ? 45 : 44); break; }
                    const uint32_t dst = tiles + stage * TILE_BYTES + (is_v ? (w4 >> 1) * (HALVES * PANEL_BYTES) : (w4 >> 1) * PANEL_BYTES);
                    uint32_t flags = 0;
#pragma unroll
                    for (int i = 0; i < TURNS; ++i) {
                        const int row = (w4 & 1) * 32 + i * AT_ONCE + r_in, key = key0 + (w4 >> 1) * 64 + row;      // row of the page
                        uint32_t* v = &codes[i].x;
                        const int e = (int)scale[i] - (int)scale0, fold = min(max(e, FOLD_LOW), FOLD_HIGH);
                        const bool live = key < key_end;
                        if (edge && is_v) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                if (!live) v[k] = 0u;
                                const uint32_t bad = no_numbers<true>(v[k]);
                                if (bad) flags |= 2u;
                                v[k] &= ~bad;
                            }
                        }
                        if (live && e != fold) flags |= 1u;
                        const __half2 by = __float2half2_rn(q3_exp2i(fold));
                        uint32_t h[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const __half2 z = __hmul2(q3_half2_of(v[k >> 1] >> (16 * (k & 1))), by);
                            h[k] = *reinterpret_cast<const uint32_t*>(&z);
                        }
                        // the lanes of a row's second half (64 values) store their second chunk first: eight lanes, eight banks
                        const int swap = HALVES == 2 ? c >> 2 : 0;
                        const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
                        const int half_bytes = is_v ? PANEL_BYTES : HALF_BYTES;
                        st_shared_v4(dst + chunk_at(row, 2 * c + swap, half_bytes), swap ? hi : lo);
                        st_shared_v4(dst + chunk_at(row, 2 * c + 1 - swap, half_bytes), swap ? lo : hi);
                    }
                    flags = __reduce_or_sync(0xffffffffu, flags);
                    // what the fold leaves, as a factor of the key's score or in log2 units: read only where a flag says so, which any warp of either kind may
                    if (c == 0) {
#pragma unroll
                        for (int i = 0; i < TURNS; ++i) {
                            const int row = w4 * 32 + i * AT_ONCE + r_in, e = (int)scale[i] - (int)scale0, rest = e - min(max(e, FOLD_LOW), FOLD_HIGH);
                            const bool live = key0 + row < key_end;                  // (the scale of a row that nobody wrote may be anything)
                            if (is_v) sh.value_rest[note][row] = live ? (float)rest : 0.0f;
                            else sh.key_rest[note][row] = live ? q3_exp2i(rest) : 1.0f;
                        }
                    }
                    Note& to_note = is_v ? sh.values[note] : sh.keys[note];
                    if (lane == 0) {
                        to_note.flags[w4] = flags;
                        if (w4 == 0) to_note.scale = is_v ? (float)((int)scale0 - Q3_SCALE_BIAS) : q3_exp2i((int)scale0 - Q3_SCALE_BIAS);
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        if (!is_v) mbar_arrive(bar_noted + 8 * note);
                        mbar_arrive(bar_full + 8 * stage);
                    }
                    if (n + 1 < steps) load(part.begin + n + 1);
                }
            } else {
                auto ask = [&](int n, int number) {                                  // the copies of a stretch, by one thread
                    const int stage = number % STAGES;
                    const uint32_t bar = (is_v ? bar_v_here : bar_k_full) + 8 * stage, dst = tiles + stage * TILE_BYTES;
                    mbar_expect_tx(bar, TILE_BYTES);
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const int row = (int)((page_of(st, table, 2 * (part.begin + n) + p) * st.nkv + part.head) * PAGE);
#pragma unroll
                        for (int h = 0; h < HALVES; ++h)
                            tma_load_2d(is_v ? dst + p * (HALVES * PANEL_BYTES) + h * PANEL_BYTES : dst + h * HALF_BYTES + p * PANEL_BYTES, is_v ? &map_v : &map_k, bar,
                                        h * 64, row);
                    }
                };
                auto stage_free = [&](int number) { return mbar_wait_warp(bar_empty + 8 * (number % STAGES), ((uint32_t)(number / STAGES) & 1u) ^ 1u); };
                for (int n = 0; n < steps && ok; ++n, ++stretch) {
                    if (w4 == 0) {
                        ok = stage_free(stretch);
                        if (!ok) { failed(is_v ? 45 : 44); break; }
                        if (lane == 0) ask(n, stretch);
                        __syncwarp();
                    }
                    if (!is_v) continue;
                    const int stage = stretch % STAGES, key0 = (part.begin + n) * STRETCH;
                    ok = mbar_wait_warp(bar_v_here + 8 * stage, (uint32_t)(stretch / STAGES) & 1u);
                    if (!ok) { failed(46); break; }
                    if (key0 + STRETCH > pos0) {
                        // values behind the end, and those that are no numbers, become zeros; a warp looks through 32 rows
                        uint32_t found = 0;
                        const uint32_t page = v_smem + stage * TILE_BYTES + (w4 >> 1) * (HALVES * PANEL_BYTES);
                        for (int i = lane; i < 32 * (D / 8); i += 32) {
                            const int row = (w4 & 1) * 32 + i / (D / 8), key = key0 + (w4 >> 1) * 64 + row;
                            const uint32_t at_chunk = page + chunk_at(row, i % (D / 8), PANEL_BYTES);
                            uint4 v = ld_shared_v4(at_chunk);
                            if (key >= key_end) v = make_uint4(0, 0, 0, 0);
                            const uint4 bad = make_uint4(no_numbers<false>(v.x), no_numbers<false>(v.y), no_numbers<false>(v.z), no_numbers<false>(v.w));
                            const uint32_t any = bad.x | bad.y | bad.z | bad.w;
                            found |= any;
                            if (any != 0 || key >= key_end) st_shared_v4(at_chunk, make_uint4(v.x & ~bad.x, v.y & ~bad.y, v.z & ~bad.z, v.w & ~bad.w));
                        }
                        found = __reduce_or_sync(0xffffffffu, found);
                        if (lane == 0) sh.values[stretch % NOTES].flags[w4] = found != 0 ? 2u : 0u;
                        fence_proxy_async();
                        __syncwarp();
                    }
                    if (lane == 0) mbar_arrive(bar_v_full + 8 * stage);
                }
            }
            at = Work::next(share, at, part);
        }
    } else {
        // ------------------------------------------------ the products: the whole warp walks and one elected thread issues
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MMA_REGS));
        if (warp == MMA_WARP) {
        constexpr uint32_t idesc_s = idesc(F8, BM, STRETCH, false), idesc_pv = idesc(F8, BM, D, true);
        const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t q_desc = desc_k_major(q_smem), k_desc = desc_k_major(k_smem), v_desc = desc_mn_major(v_smem, PANEL_BYTES);
        int stretch = 0;
        uint32_t q_turn = 0, turn[2] = {0, 0}, done[2] = {0, 0};                    // parities: queries, weights of a tile, products of a tile
        bool ok = true;
        auto scores = [&](int x, int number, bool release) {
            const uint32_t stage = (uint32_t)number % STAGES;
            const uint64_t q_src = q_desc + (uint64_t)(x * (TILE_BYTES >> 4)), k_src = k_desc + (uint64_t)(stage * (TILE_BYTES >> 4));
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (kk >> 2) * HALF_BYTES + (kk & 3) * 32;
                    tc_mma_ss(acc + COL_S + x * 128, q_src + (uint64_t)(off >> 4), k_src + (uint64_t)(off >> 4), idesc_s, kk > 0 ? 1u : 0u);
                }
                tc_commit(bar_s_full + 8 * x);
                if (release) tc_commit(bar_k_empty + 8 * stage);
            }
            __syncwarp();
        };
        for (int at = share.from; at < share.to && ok;) {
            const TreePart part = Work::part(st, share, at, blockIdx.x);
            const int rows = Work::n_new(st, part.seq) * group - part.tile * ROWS, steps = part.end - part.begin, both = rows > BM ? 2 : 1;
            auto keys_here = [&](int number) { return mbar_wait_warp(bar_k_full + 8 * (number % STAGES), (uint32_t)(number / STAGES) & 1u); };
            ok = mbar_wait_warp(bar_q, q_turn) && keys_here(stretch);
            q_turn ^= 1u;
            if (!ok) { failed(47); break; }
            tc_fence_after();
            for (int x = 0; x < both; ++x) scores(x, stretch, x == both - 1);
            for (int i = 0; i < steps && ok; ++i, ++stretch) {
                for (int x = 0; x < both && ok; ++x) {
                    const uint32_t stage = (uint32_t)stretch % STAGES;
                    ok = mbar_wait_warp(bar_p_full + 8 * x, turn[x]) && mbar_wait_warp(bar_v_full + 8 * stage, (uint32_t)(stretch / STAGES) & 1u);
                    turn[x] ^= 1u;
                    if (!ok) { failed(48); break; }
                    tc_fence_after();
                    const uint64_t v_src = v_desc + (uint64_t)(stage * (TILE_BYTES >> 4));
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < STRETCH / 16; ++kk) {
                            const uint32_t off = (kk >> 2) * (HALVES * PANEL_BYTES) + (kk & 3) * 16 * 128;
                            tc_mma_ts(acc + COL_O + x * 128, acc + COL_S + x * 128 + kk * 8, v_src + (uint64_t)(off >> 4), idesc_pv, (i > 0 || kk > 0) ? 1u : 0u);
                        }
                        tc_commit(bar_pv_done + 8 * x);
                        if (x == both - 1) tc_commit(bar_v_empty + 8 * stage);
                    }
                    __syncwarp();
                    // the next scores go where the weights were: once the products with them are done
                    ok = mbar_wait_warp(bar_pv_done + 8 * x, done[x]);
                    done[x] ^= 1u;
                    if (ok && i + 1 < steps) {
                        ok = keys_here(stretch + 1);
                        if (ok) {
                            tc_fence_after();
                            scores(x, stretch + 1, x == both - 1);
                        }
                    }
                    if (!ok) failed(49);
                }
            }
            at = Work::next(share, at, part);
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---- the parts of the items that several blocks share, added up in their order: for every block of the first kernel whose last part is the first one of such
// an item, and for 32 of its rows, a block
__global__ void __launch_bounds__(256) tree_tc_merge_kernel(const __grid_constant__ Args a, int blocks) {
    __shared__ TreeShare shared_share;
    pdl_launch_dependents();
    pdl_wait();
    const TreeStep& st = a.step;
    const int b0 = blockIdx.x;
    if (threadIdx.x < 32) {
        const TreeShare found = Work::share(st, 1, b0, blocks);
        if (threadIdx.x == 0) shared_share = found;
    }
    __syncthreads();
    TreeShare share = shared_share;
    if (share.from >= share.to) return;
    TreePart part;
    for (int at = share.from; at < share.to; at = Work::next(share, at, part)) part = Work::part(st, share, at, b0);
    if (part.parts == 1 || part.begin != 0) return;
    const int group = st.nq / st.nkv, t0 = st.seq_start[part.seq], n_new = Work::n_new(st, part.seq);
    const int row0 = part.tile * ROWS, rows = min(ROWS, n_new * group - row0), first = blockIdx.y * 32;
    if (first >= rows) return;
    const int r = first + (threadIdx.x & 31);
    if (r >= rows) return;
    bf16* const out = a.out + ((int64_t)(t0 + (row0 + r) / group) * st.nq + part.head * group + (row0 + r) % group) * D;
    for (int c = threadIdx.x >> 5; c < D / 8; c += 8) {                              // eight values a turn
        float m = -INFINITY, l = 0.0f, v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        for (int b = 0; b < part.parts; ++b) {
            const float* src = a.parts + (int64_t)part.slot_of(b) * PART;
            const float2 ml = *reinterpret_cast<const float2*>(src + ROWS * D + 2 * r);
            const float4 u0 = *reinterpret_cast<const float4*>(src + ((2 * c) * ROWS + r) * 4), u1 = *reinterpret_cast<const float4*>(src + ((2 * c + 1) * ROWS + r) * 4);
            const float m2 = fmaxf(m, ml.x), was = m == m2 ? 1.0f : ex2(m - m2), now = ml.x == m2 ? 1.0f : ex2(ml.x - m2);
            m = m2;
            l = fmaf(now, ml.y, l * was);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = fmaf(now, (&u0.x)[e], v[e] * was);
                v[e + 4] = fmaf(now, (&u1.x)[e], v[e + 4] * was);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint4 w;
        w.x = pack2<false>(v[0] * inv, v[1] * inv);
        w.y = pack2<false>(v[2] * inv, v[3] * inv);
        w.z = pack2<false>(v[4] * inv, v[5] * inv);
        w.w = pack2<false>(v[6] * inv, v[7] * inv);
        *reinterpret_cast<uint4*>(out + 8 * c) = w;
    }
}

template <bool F8> int launch(const Args& a, int max_new, cudaStream_t stream) {
    static Q3PerDevice configured;
    const cudaError_t e = q3_allow_shared_memory(tree_tc_kernel<F8>, SMEM_BYTES, configured);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_k = {}, map_v = {};
    if (!F8 && (!q3_make_map_bf16(&map_k, a.keys, a.step.n_pages * a.step.nkv * PAGE, D, PAGE, 64, true) ||
                !q3_make_map_bf16(&map_v, a.values, a.step.n_pages * a.step.nkv * PAGE, D, PAGE, 64, true)))
        return Q3_ERR_BAD_SIZE;
    const int64_t units = Work::most_units(a.step);
    if (units > 0x3fffffff) return Q3_ERR_TOO_LARGE;
    const int sms = q3_device_sm_count(), blocks = (int)(units < sms ? units : sms);
    int code = (int)q3_launch(tree_tc_kernel<F8>, dim3(blocks), dim3(THREADS), (size_t)SMEM_BYTES, stream, map_k, map_v, a);
    if (code != 0) return code;
    const int rows = (int64_t)max_new * (a.step.nq / a.step.nkv) < ROWS ? max_new * (a.step.nq / a.step.nkv) : ROWS;
    return (int)q3_launch(tree_tc_merge_kernel, dim3(blocks, (rows + 31) / 32), dim3(256), 0, stream, a, blocks);
}

}  // namespace

Q3_EXPORT int q3_attention_tree_tc_head_dim() { return D; }

// Float32 values of `parts` for a launch.
Q3_EXPORT int64_t q3_attention_tree_tc_parts() { return (int64_t)2 * q3_device_sm_count() * PART; }

Q3_EXPORT int q3_attention_tree_tc_bf16(const void* q, const void* k_pages, const void* v_pages, const void* k_scales, const void* v_scales,
                                        void* out, float* parts, const int* seq_start, const int* seq_pos0, const int* page_table,
                                        int pages_per_seq, int64_t n_pages, int n_seqs, int max_new, int nq, int nkv, float scale,
                                        const void* tree, int words, int* status, void* stream) {
    if (n_seqs <= 0 || max_new <= 0) return 0;
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || n_pages <= 0 || pages_per_seq <= 0 || !(scale > 0.0f) || (tree != nullptr && (words <= 0 || words * 64 < max_new)))
        return Q3_ERR_BAD_SIZE;                                                      // (the maximum is taken before the scale)
    if (n_pages * nkv * PAGE > 0x7fffffff) return Q3_ERR_TOO_LARGE;                  // a row's number is a coordinate of a copy
    if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) || !aligned16(parts)) return Q3_ERR_MISALIGNED;
    const Args a = {{seq_start, seq_pos0, page_table, (const unsigned long long*)tree, words, pages_per_seq, n_seqs, nq, nkv, n_pages, max_new},
                    (const bf16*)q, (bf16*)out, (const unsigned char*)k_pages, (const unsigned char*)v_pages, (const uint8_t*)k_scales,
                    (const uint8_t*)v_scales, parts, status, scale * 1.4426950408889634f};
    return k_scales != nullptr ? launch<true>(a, max_new, (cudaStream_t)stream) : launch<false>(a, max_new, (cudaStream_t)stream);
}
