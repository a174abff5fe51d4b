// Attention of a step's new tokens over the cache's pages in bfloat16 or in 8 bits on the 5th-generation tensor cores, for trees (or runs) whose
// rows - a row is a token and a query head - fill tiles of 128.  What a token sees and what comes out is said in attention_tree.cu.
//
// S = Q K^T and O += P V are tcgen05.mma over a page of 64 keys, with the accumulators and the weights in tensor memory.  A tile has two buffers of scores there, so
// that a page's scores are made while the softmax is at the page before: its chain is then the softmax alone.  (With the queries in tensor memory, which leaves
// room for one buffer, products of 128 x 64 x 16 take 33 cycles instead of 51, but scores wait for the products before them: 2,750 cycles a page against 2,200.)
// A block, one an SM, works on two tiles side by side, so that the products of one run under the softmax of the other:
//   more than 128 rows   two tiles of 128 rows, which take the same pages;
//   up to 128 rows       twice the same rows, one tile with the pages of even number and one with those of odd number; their sums meet at the end.
// The pages of all items are shared out evenly over the blocks (tree_work.cuh).
//   warps 0-7    softmax: thread r of a tile's 128 owns row r (TMEM lane r).  It brings in its query, reads its 64 scores, writes the weights over them, and
//                rescales O when the maximum is raised by more than 2^8.  At the end of a part it writes the row, or its share of it for the second
//                kernel to add up.
//   warps 8-15   8 bits: turn the codes of keys (8-11) and values (12-15) into half precision, which holds them exactly, where TMA would have put them;
//                bfloat16: 12-15 look through the values of the pages that some row does not see in whole.
//   warps 16, 19 issue the products, one elected thread of each those of a tile.
//   warps 17, 18 copy keys and values: bfloat16 by TMA where the products read them, 8 bits as they lie, some pages ahead.
//
// 8 bits.  A page's keys are brought to one scale, that of its first row, 2^k0, by folding 2^(k - k0) into the half-precision numbers, which is exact
// for k - k0 in -14 .. 7; so are its values, to the largest scale 2^v0 of its rows that all tokens see.  Scores are then multiplied by 2^k0 with the softmax's own scale; v0 is added to the scores
// in log2 units, so that a weight is w = 2^(x + v0 - M) with M the running maximum of x + v0 and the sum of the softmax that of w 2^-v0.  The largest term's weight is not
// below 2^-14 of M, since its value is folded by no more (2^-21 where a new token's scale is above 2^v0), and half precision drops what is below 2^-31 of M.  Where some row of a page has a scale outside that
// range, what is missing (`rest`) is added score by score, in a path of its own.  Queries are brought into half precision as in attention_tree_mma.cu.
//
// A value that is no number (infinity, NaN) in a page that some row does not see in whole is taken out before the product, and put into the
// outputs of the rows that see it: 0 times a NaN would reach the others.
// What bounds it: a page and 256 rows are 1,340 cycles of the tensor pipe (products of 128 x 64 x 16 from shared memory take 51 cycles, those with the weights
// 65) and 1,024 of the special-function unit (an exponential a score), but 2,200 pass in bfloat16 and 3,000 in 8 bits: the softmax's chain of a page and that of
// the products' warp are each as long, seven waits of 130 to 160 cycles and what lies between.  (Without any exponential it takes 5 % less, with an eighth of
// the products 15 %; two sets of softmax warps that take turns, or products of keys and of values by warps of their own: within 3 %.)  Beginning and ending a
// part are 16,000 cycles.  1 sequence of 32,000 keys, 33 tokens and 64 heads over 8 (bfloat16) 70 us, the floor being 21; 8 of up to 8,000, 64 and 40 (8 bits)
// 94 (22); 8 of up to 3,000, 7 and 32 (bfloat16) 27.5 (11).
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
static_assert(PAGE == 64, "a product takes a page of 64 keys");
constexpr int BM = 128, ROWS = 2 * BM, HALVES = D / 64;
constexpr int SOFTMAX_WARPS = 8, TURN_WARPS = 4, V_WARP = 12, MMA_WARP = 16, K_COPY_WARP = 17, V_COPY_WARP = 18, THREADS = 20 * 32;
// Registers of a thread by role: 256 x 144 + 256 x 72 + 128 x 48 = 640 x 96, what the block is launched with.
constexpr int LAUNCH_REGS = 96, SOFTMAX_REGS = 144, TURN_REGS = 72, MMA_REGS = 48;
static_assert(8 * 32 * SOFTMAX_REGS + 8 * 32 * TURN_REGS + 4 * 32 * MMA_REGS <= THREADS * LAUNCH_REGS, "shares of the launch's registers");
constexpr int NOTES = 8;                                  // pages whose notes are kept: more than lie between the copies and the softmax
constexpr int PANEL_BYTES = PAGE * 128, TILE_BYTES = HALVES * PANEL_BYTES;                 // 64 rows of 128 bytes; a page's keys or values in 16 bits
constexpr int CODE_BYTES = PAGE * D;
constexpr uint32_t TMEM_COLS = 512, TILE_COLS = 256, COL_S = 0, COL_O = 128;              // of tile x, from x * 256 on; two buffers of S, P lies over S
constexpr int Q_BYTES = HALVES * BM * 128, MEET_COLS = D / 2;                             // a tile's queries; columns of the sums that meet at a time
static_assert(BM * MEET_COLS * 4 <= Q_BYTES, "they meet where the second tile's queries would be");
// Pages that take about as long as beginning and ending a part.  0 / 3 / 6 / 9: 32 sequences of up to 4,000 keys and 32 new tokens (bfloat16) 129 / 93 / 78 /
// 76 us, 8 of up to 8,000 and 64 (8 bits) 118 / 100 / 95 / 99; as much longer a piece may be: 12 of up to 5,000 and 12 (bfloat16) 45 with 6, 57 with 40.
constexpr int PART_PAGES = 6;
// A block is given no fewer pages; in the time of how many pages a part is added up: 0 / 0.05 / 0.12 / 0.25 for 1 sequence of 32,000 keys of one kv head, 20 tokens
// and 8 heads 55 / 50 / 43 / 40 us, 2 of up to 30,000 and 24 (8 bits) 57 / 53 / 48 / 45, of up to 3,000 of 8 kv heads and 8 18.7 / 18.5 / 18.5 / 19.3.
constexpr int LEAST_PAGES = 2;
constexpr float JOIN_PAGES = 0.2f;
constexpr float RAISE = 8.0f, LIFT = 6.0f;                // 8 bits: weights are this much larger (in log2), up to 2^14, and lose nothing above 2^-20 of M
constexpr int FOLD_LOW = -14, FOLD_HIGH = 7;
constexpr int PART = ROWS * (D + 2);                      // float32 of a part: sums [D / 4][ROWS][4], then (maximum, sum) [ROWS][2]
// An item of several parts, the first of which is a block's last: noted behind all parts, a note a block, for the second kernel (parts 0: there is none).
struct MergeNote {
    int parts, slot0, first_block, rows, first_row, t0, head, pad;
};
static_assert(sizeof(MergeNote) == 32, "eight words");

struct Note {                                             // what is noted of a page
    float scale;                                          // 8 bits: 2^k0 (values: v0)
    uint32_t flags[TURN_WARPS];                           // bit 0: some scale is out of range; bit 1: some value is no number (8 bits: the first two words)
    uint32_t pad[3];
};
template <bool F8> struct Layout {
    static constexpr int STAGES = F8 ? 2 : 4;             // pages of keys and of values that the products can read
    static constexpr int CODES = F8 ? 4 : 0;              // pages of codes of either on their way: what a page's copy takes, some 3,500 cycles, has to go by
    static constexpr int QUERIES = 0, MEET = Q_BYTES, K = 2 * Q_BYTES, V = K + STAGES * TILE_BYTES;
    static constexpr int K_CODES = V + STAGES * TILE_BYTES, V_CODES = K_CODES + CODES * CODE_BYTES, REST = V_CODES + CODES * CODE_BYTES;
    // barriers: one word of 8 bytes each
    static constexpr int Q = 0, S_FULL = 1, P_FULL = 5, PV_DONE = 9, NOTED = 11, K_FULL = NOTED + NOTES, K_EMPTY = K_FULL + STAGES, V_FULL = K_EMPTY + STAGES;
    static constexpr int V_EMPTY = V_FULL + STAGES, V_HERE = V_EMPTY + STAGES;             // V_HERE: TMA's values, before they are looked through
    static constexpr int KC_FULL = V_HERE + STAGES, KC_EMPTY = KC_FULL + CODES, VC_FULL = KC_EMPTY + CODES, VC_EMPTY = VC_FULL + CODES;
    static constexpr int MET = VC_EMPTY + CODES, MET_FREE = MET + 1, BARS = MET + 2;       // the sums of odd pages lie in MEET; they are read
};
template <bool F8> struct Shared {
    uint8_t code_scales[2][F8 ? Layout<F8>::CODES : 1][PAGE];
    Note keys[NOTES], values[NOTES];
    float key_rest[NOTES][PAGE], value_rest[NOTES][PAGE];
    float2 meet[BM];                                      // (maximum, sum) of a tile of odd pages
    TreeShare share;
    TreePart part;
    unsigned long long bars[Layout<F8>::BARS];
    uint32_t tmem;
};
template <bool F8> constexpr int smem_bytes = Layout<F8>::REST + (int)sizeof(Shared<F8>);
static_assert(smem_bytes<true> <= 227 * 1024 && smem_bytes<false> <= 227 * 1024, "shared memory of a block");

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

using Work = TreeWork<PAGE, ROWS, true>;

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
__device__ __forceinline__ void load_words2(uint32_t* w, uint32_t at) {
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
}
// 16-byte chunk `c` (of D / 8) of row r of a tile whose halves of 64 columns are `half_bytes` apart, as TMA's 128-byte swizzle lays it.
__device__ __forceinline__ uint32_t chunk_at(int r, int c, int half_bytes) { return (uint32_t)((c >> 3) * half_bytes + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// A page number of a sequence, within the cache whatever the table says.
__device__ __forceinline__ int64_t page_of(const TreeStep& st, const int* table, int i) {
    const int p = i < st.pages_per_seq ? table[i] : 0;
    return p >= 0 && p < st.n_pages ? p : 0;
}

// Bytes from global memory as they lie (all a multiple of 16).
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Where the values of an output row are that are no numbers: bit d of `plus` for +infinity, of `minus` for -infinity, of both for NaN.
struct Odd {
    uint32_t plus[D / 32], minus[D / 32];
    bool any;
};

// The values of page `s` that are no numbers, of the keys that the row sees.
template <bool F8>
__device__ __noinline__ void find_odd(const Args& a, const int* table, int head, int s, unsigned long long seen, Odd& odd) {
    for (int key = 0; key < PAGE; ++key) {
        if (!(seen >> key & 1)) continue;
        const int64_t cell = (page_of(a.step, table, s) * a.step.nkv + head) * PAGE + key;
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
    using L = Layout<F8>;
    extern __shared__ unsigned char smem[];
    pdl_launch_dependents();
    const uint32_t base = smem_u32(smem);
    Shared<F8>& sh = *reinterpret_cast<Shared<F8>*>(smem + L::REST);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bars = smem_u32(sh.bars);
    auto bar = [&](int which, int i) { return bars + 8 * (which + i); };
    if (base & 1023u) {                                  // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) atomicExch(a.status, 40);
        return;
    }
    if (threadIdx.x == 0) {
        mbar_init(bar(L::Q, 0), SOFTMAX_WARPS + 2);      // (with the warps that wait for it: it cannot be two parts ahead of them)
        mbar_init(bar(L::MET, 0), 4);
        mbar_init(bar(L::MET_FREE, 0), 4);
        for (int x = 0; x < 2; ++x) {
            for (int b = 0; b < 2; ++b) {                // of a tile's two buffers
                mbar_init(bar(L::S_FULL, 2 * x + b), 1);
                mbar_init(bar(L::P_FULL, 2 * x + b), 4);
            }
            mbar_init(bar(L::PV_DONE, x), 1);
        }
        for (int n = 0; n < NOTES; ++n) mbar_init(bar(L::NOTED, n), TURN_WARPS);
        for (int s = 0; s < L::STAGES; ++s) {
            mbar_init(bar(L::K_FULL, s), F8 ? 2 : 1);
            mbar_init(bar(L::K_EMPTY, s), 2);
            mbar_init(bar(L::V_FULL, s), F8 ? 2 : TURN_WARPS);
            mbar_init(bar(L::V_EMPTY, s), 2);
            mbar_init(bar(L::V_HERE, s), 1);
        }
        for (int s = 0; s < L::CODES; ++s) {
            mbar_init(bar(L::KC_FULL, s), 1);
            mbar_init(bar(L::KC_EMPTY, s), 2);
            mbar_init(bar(L::VC_FULL, s), 1);
            mbar_init(bar(L::VC_EMPTY, s), 2);
        }
        mbar_init_fence();
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    const TreeStep& st = a.step;
    if (warp == 0) {
        // the first part is found by this warp for all (most blocks have no other): 4,000 cycles for each role by itself
        TreeShare found = Work::share(st, LEAST_PAGES, LEAST_PAGES, JOIN_PAGES, PART_PAGES, blockIdx.x, gridDim.x);
        TreePart first = {};
        if (found.from < found.to) first = Work::part(st, found, found.from, blockIdx.x);
        if (lane == 0) {
            sh.share = found;
            sh.part = first;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    TreeShare share = sh.share;
    const int group = st.nq / st.nkv;
    auto failed = [&](int where) { if (lane == 0) atomicExch(a.status, where); };
    // The turn of a barrier whose phases are pages, `number` of them in a ring of `size`.
    auto turn_of = [](int number, int size) { return (uint32_t)(number / size) & 1u; };

    if (warp < SOFTMAX_WARPS) {
        // ------------------------------------------------ softmax: thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        const int x = warp >> 2, r = (warp & 3) * 32 + lane;                         // tile, row of it
        const uint32_t t_tile = tmem + ((uint32_t)((warp & 3) * 32) << 16) + x * TILE_COLS;
        int page0 = 0;                                                               // pages of this block before the part
        MergeNote merge = {};
        uint32_t count = 0, q_turn = 0, met_turn = 0;                                // pages of this tile so far; parities of the parts, of the tiles' meetings
        bool ok = true;
        for (int at = share.from; at < share.to && ok;) {
            const TreePart part = at == share.from ? sh.part : Work::part(st, share, at, blockIdx.x);
            if (part.begin >= part.end) break;
            const int t0 = part.t0, n_new = part.n_new, pos0 = part.pos0;
            const int all_rows = n_new * group - part.tile * ROWS, steps = part.end - part.begin;
            const bool split = all_rows <= BM;                                       // one tile of rows: every other page
            const int first = split ? x : 0, stride = split ? 2 : 1;
            const int rows = split ? all_rows : all_rows - x * BM, row = part.tile * ROWS + (split ? 0 : x * BM) + r, own = min(row / group, n_new - 1);
            const int64_t row_at = ((int64_t)(t0 + own) * st.nq + part.head * group + row % group) * D;
            // ---- the warp's queries, D / 8 lanes a row, each 16 bytes (twice the same rows: both tiles' products read the first one's, but the second one's
            // warps want the rows' factors too).  In loops that are not unrolled: this is run once a part, from instructions that have left the caches by then.
            float factor = a.scale_log2;
            {
                constexpr int PER_ROW = D / 8, AT_ONCE = 32 / PER_ROW, TURNS = 32 / AT_ONCE;
                const int c = lane % PER_ROW;
                const uint32_t queries = base + L::QUERIES + x * Q_BYTES;
                __syncwarp();
#pragma unroll 1
                for (int i = 0; i < TURNS; ++i) {
                    const int of = i * AT_ONCE + lane / PER_ROW, to_row = (warp & 3) * 32 + of;       // the lane whose row this is
                    const int64_t from = __shfl_sync(0xffffffffu, row_at, of);
                    const uint32_t dst = queries + chunk_at(to_row, c, BM * 128);
                    if (to_row < rows) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(a.q + from + 8 * c) : "memory");
                    else st_shared_v4(dst, make_uint4(0, 0, 0, 0));
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if constexpr (F8) {
                    // a row's numbers by one power of two into half precision, each thread its own row
                    __syncwarp();
                    uint32_t tops = 0;
#pragma unroll 4
                    for (int i = 0; i < PER_ROW; ++i) {
                        const uint4 w = ld_shared_v4(queries + chunk_at(r, i, BM * 128));
                        tops = __vmaxu2(tops, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
                    }
                    int e2 = (int)(max(tops & 0xffffu, tops >> 16) >> 7) - 127;
                    e2 = e2 >= 128 ? 0 : min(max(e2, -60), 60);
                    const float down = q3_exp2i(-e2);
                    factor *= q3_exp2i(e2);
#pragma unroll 4
                    for (int i = 0; i < PER_ROW; ++i) {
                        const uint32_t at_chunk = queries + chunk_at(r, i, BM * 128);
                        uint4 w = ld_shared_v4(at_chunk);
                        uint32_t* v = &w.x;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = pack2<true>(__uint_as_float(v[e] << 16) * down, __uint_as_float(v[e] & 0xffff0000u) * down);
                        st_shared_v4(at_chunk, w);
                    }
                }
                fence_proxy_async();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(L::Q, 0));

            float m_run = -INFINITY, l_run = 0.0f;
            Odd odd;
            odd.any = false;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) odd.plus[i] = odd.minus[i] = 0u;
            for (int n = first; n < steps; n += stride, ++count) {
                const int key0 = (part.begin + n) * PAGE, number = page0 + n, note = number % NOTES;
                const uint32_t buffer = count & 1u, turn = count >> 1 & 1u, t_s = t_tile + COL_S + buffer * 64;
                const bool edge = key0 + PAGE > pos0;                                // some key is a new token's, or behind the end
                ok = mbar_wait_warp(bar(L::S_FULL, 2 * x + buffer), turn);
                if (!ok) { failed(41); break; }
                if (F8 || edge) {
                    ok = mbar_wait_warp(bar(L::NOTED, note), turn_of(number, NOTES));
                    if (!ok) { failed(42); break; }
                }
                tc_fence_after();
                // ---- of the page: score = dot * c1, in log2 units, and v0
                float c1 = factor, v0 = 0.0f;
                bool rests = false;
                if constexpr (F8) {
                    c1 = fmaxf(c1 * sh.keys[note].scale, 1.2e-38f);                  // (what is not seen stays minus infinity)
                    v0 = sh.values[note].scale;
                    rests = (sh.keys[note].flags[0] | sh.keys[note].flags[1] | sh.values[note].flags[0] | sh.values[note].flags[1]) & 1u;
                }
                if (edge) {
                    // scores of keys that the row does not see become minus infinity where they lie
                    const unsigned long long* mask = st.tree != nullptr ? st.tree + (int64_t)(t0 + own) * st.words : nullptr;
                    const unsigned long long seen = tree_seen(mask, st.words, pos0, n_new, own, key0);
                    uint32_t flags = sh.values[note].flags[0] | sh.values[note].flags[1];
                    if constexpr (!F8) flags |= sh.values[note].flags[2] | sh.values[note].flags[3];
                    if (flags & 2u) find_odd<F8>(a, st.page_table + (int64_t)part.seq * st.pages_per_seq, part.head, part.begin + n, seen, odd);
                    __syncwarp();
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        uint32_t s[32];
                        const uint32_t bits = (uint32_t)(seen >> (32 * h));
                        tc_ld32(t_s + 32 * h, s);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!(bits >> e & 1u)) s[e] = 0xff800000u;
                        tc_st32(t_s + 32 * h, s);
                    }
                    tc_wait_st();
                }
                // ---- the maximum of x + v0 (and the rests)
                float top;
                if (F8 && rests) {
                    top = -INFINITY;
#pragma unroll 1
                    for (int h = 0; h < 2; ++h) {
                        uint32_t s[32];
                        tc_ld32(t_s + 32 * h, s);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) top = fmaxf(top, fmaf(__uint_as_float(s[e]) * sh.key_rest[note][32 * h + e], c1, sh.value_rest[note][32 * h + e]));
                    }
                } else {
                    uint32_t s[64];
                    tc_ld32(t_s, s);
                    tc_ld32(t_s + 32, s + 32);
                    tc_wait_ld();
                    float mx[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 4]));
#pragma unroll
                    for (int e = 8; e < 64; e += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mx[k] = max3(mx[k], __uint_as_float(s[e + k]), __uint_as_float(s[e + k + 4]));
                    top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c1;
                }
                top += v0;
                const bool raise = top > m_run + RAISE;
                float alpha = 1.0f;
                if (raise) {
                    alpha = ex2(m_run - top);
                    m_run = top;
                    l_run *= alpha;
                }
                // ---- weights, over the scores
                const float shift = v0 - (m_run == -INFINITY ? 0.0f : m_run) + (F8 ? LIFT : 0.0f);
                const float2 c2 = make_float2(c1, c1), shift2 = make_float2(shift, shift);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                __syncwarp();
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    uint32_t s[32], p[16];
                    tc_ld32(t_s + 32 * h, s);
                    tc_wait_ld();
                    if (F8 && rests) {
                        // (where nothing is left by the folds, these are the other path's numbers to the bit: a row does not feel the scales of
                        // keys that it does not see)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float w[2];
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const float rest = sh.value_rest[note][32 * h + e + k];
                                w[k] = ex2(fmaf(__uint_as_float(s[e + k]) * sh.key_rest[note][32 * h + e + k], c1, shift + rest));
                                float& to_sum = k == 0 ? sum[(e >> 1) & 1].x : sum[(e >> 1) & 1].y;
                                to_sum = fmaf(w[k], ex2(-rest), to_sum);
                            }
                            p[e / 2] = pack2<true>(w[0], w[1]);
                        }
                        __syncwarp();
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 z = __ffma2_rn(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), c2, shift2);
                            const float2 w = make_float2(ex2(z.x), ex2(z.y));
                            sum[(e >> 1) & 1] = __fadd2_rn(sum[(e >> 1) & 1], w);
                            p[e / 2] = pack2<F8>(w.x, w.y);
                        }
                    }
                    tc_st16(t_s + 16 * h, p);
                }
                const float total = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                l_run += F8 ? total * ex2(-v0) : total;
                // the products of the page before have to be done where O is rescaled, and once the part ends: this page's are waited for then, and a
                // parity tells a phase from the next one, not from the one after that
                const bool rescale = n > first && __any_sync(0xffffffffu, raise);
                if (rescale || (n > first && n + stride >= steps)) {
                    ok = mbar_wait_warp(bar(L::PV_DONE, x), (count - 1) & 1u);
                    if (!ok) { failed(37); break; }
                    tc_fence_after();
                }
                if (rescale) {
#pragma unroll 1
                    for (int c = 0; c < D; c += 64) {
                        uint32_t s[64];
                        tc_ld32(t_tile + COL_O + c, s);
                        tc_ld32(t_tile + COL_O + c + 32, s + 32);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 64; ++e) s[e] = __float_as_uint(__uint_as_float(s[e]) * alpha);
                        tc_st32(t_tile + COL_O + c, s);
                        tc_st32(t_tile + COL_O + c + 32, s + 32);
                    }
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(L::P_FULL, 2 * x + buffer));
            }
            if (!ok) break;
            // the part's last products; a tile without pages goes on with the other one's warps, not ahead of them
            ok = first < steps ? mbar_wait_warp(bar(L::PV_DONE, x), (count - 1) & 1u) : mbar_wait_warp(bar(L::Q, 0), q_turn);
            q_turn ^= 1u;
            if (!ok) { failed(43); break; }
            tc_fence_after();
            // ---- the row, or its part of it
            const bool whole = part.parts == 1;
            float* const dst = a.parts + (int64_t)part.slot * PART;
            const int part_row = split ? r : x * BM + r;
            float mine = 1.0f, other = 0.0f;                                         // factors of the two tiles' sums
            float4* const meet = reinterpret_cast<float4*>(smem + L::MEET);          // [MEET_COLS / 4][BM]
            if (split && x == 1) sh.meet[r] = make_float2(m_run, l_run);
            const bool here = (warp & 3) * 32 < rows;                                // some row of the warp's is one
            float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += MEET_COLS) {
                if (split) {
                    ok = x == 1 ? mbar_wait_warp(bar(L::MET_FREE, 0), met_turn ^ 1u) : mbar_wait_warp(bar(L::MET, 0), met_turn);
                    if (!ok) { failed(38); break; }
                    if (x == 0 && c0 == 0) {
                        const float2 ml = sh.meet[r];
                        const float m = fmaxf(m_run, ml.x);
                        mine = m_run == m ? 1.0f : ex2(m_run - m);
                        other = ml.x == m ? 1.0f : ex2(ml.x - m);
                        m_run = m;
                        l_run = fmaf(ml.y, other, l_run * mine);
                        inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
                    }
                }
                if (here && !(split && x == 1 && steps == 1)) {
#pragma unroll 1
                    for (int c = c0; c < c0 + MEET_COLS; c += 32) {
                        uint32_t o[32];
                        __syncwarp();
                        tc_ld32(t_tile + COL_O + c, o);
                        tc_wait_ld();
                        if (odd.any) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                if (odd.plus[c / 32] >> e & 1u) o[e] = __float_as_uint(__uint_as_float(o[e]) + INFINITY);
                                if (odd.minus[c / 32] >> e & 1u) o[e] = __float_as_uint(__uint_as_float(o[e]) - INFINITY);
                            }
                        }
                        if (split && x == 1) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4)
                                meet[(c - c0 + e) / 4 * BM + r] =
                                    make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                            continue;
                        }
                        if (split && steps > 1) {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 u = meet[(c - c0 + e) / 4 * BM + r];
                                o[e] = __float_as_uint(fmaf(u.x, other, __uint_as_float(o[e]) * mine));
                                o[e + 1] = __float_as_uint(fmaf(u.y, other, __uint_as_float(o[e + 1]) * mine));
                                o[e + 2] = __float_as_uint(fmaf(u.z, other, __uint_as_float(o[e + 2]) * mine));
                                o[e + 3] = __float_as_uint(fmaf(u.w, other, __uint_as_float(o[e + 3]) * mine));
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
                                    *reinterpret_cast<uint4*>(a.out + row_at + c + e) = v;
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 32; e += 4)
                                    *reinterpret_cast<uint4*>(dst + ((c + e) / 4 * ROWS + part_row) * 4) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                            }
                        }
                    }
                }
                if (split) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(x == 1 ? L::MET : L::MET_FREE, 0));
                    met_turn ^= 1u;
                }
            }
            if (!ok) break;
            if (split && x == 1) {                                                   // all is read: queries may come here again
                ok = mbar_wait_warp(bar(L::MET_FREE, 0), met_turn ^ 1u);
                if (!ok) { failed(39); break; }
            }
            if (!whole && r < rows && !(split && x == 1)) *reinterpret_cast<float2*>(dst + ROWS * D + 2 * part_row) = make_float2(m_run, l_run);
            tc_fence_before();
            if (!whole && part.begin == 0) merge = {part.parts, part.slot0, part.first_block, min(all_rows, ROWS), part.tile * ROWS, t0, part.head, 0};
            page0 += steps;
            at = Work::next(part);
        }
        if (threadIdx.x == 0) reinterpret_cast<MergeNote*>(a.parts + (int64_t)2 * gridDim.x * PART)[blockIdx.x] = merge;
    } else if (warp < MMA_WARP) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TURN_REGS));
        const bool is_v = warp >= V_WARP;
        const int w4 = warp & 3;
        int page0 = 0;                                                               // pages of this block before the part
        bool ok = true;
        for (int at = share.from; at < share.to && ok;) {
            const TreePart part = at == share.from ? sh.part : Work::part(st, share, at, blockIdx.x);
            if (part.begin >= part.end) break;
            const int pos0 = part.pos0, key_end = pos0 + part.n_new, steps = part.end - part.begin;
            if constexpr (F8) {
                // ------------------------------------------------ codes to half precision, a page two warps, each 32 rows of it, D / 16 lanes a row: 25
                // instructions for a lane's sixteen codes
                constexpr int PER_ROW = D / 16, AT_ONCE = 32 / PER_ROW, TURNS = 32 / AT_ONCE;
                const int c = lane % PER_ROW, r_in = lane / PER_ROW, my_stage = w4 >> 1, half = w4 & 1;
                const int full = is_v ? L::V_FULL : L::K_FULL, empty = is_v ? L::V_EMPTY : L::K_EMPTY;
                const int c_full = is_v ? L::VC_FULL : L::KC_FULL, c_empty = is_v ? L::VC_EMPTY : L::KC_EMPTY;
                // the lanes of a row's second half (64 values) take their second eight codes first: eight lanes store to eight banks
                const int swap = HALVES == 2 ? c >> 2 : 0;
                uint32_t to[2][2];                                                   // where a lane's chunks go, of rows r_in and r_in + AT_ONCE (they alternate)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        to[i][k] = base + (is_v ? L::V : L::K) + my_stage * TILE_BYTES + half * 32 * 128 +
                                   chunk_at(i * AT_ONCE + r_in, 2 * c + (k ^ swap), PANEL_BYTES) - i * AT_ONCE * 128;
                // A stage, and so the slots of its codes, are always the same warps': a barrier's parity would not tell others how far the pages between are
                static_assert(L::STAGES == 2 && L::CODES % 2 == 0 && TURN_WARPS == 4, "two warps a stage");
                for (int n = (my_stage ^ page0) & 1; n < steps; n += 2) {
                    const int number = page0 + n, slot = number % L::CODES, note = number % NOTES, key0 = (part.begin + n) * PAGE;
                    const bool edge = key0 + PAGE > pos0;
                    // The notes of values are there before their stage is: the softmax of a page does not wait for the products of two pages before.
                    // (Those of keys could then be written over ones that are still read.)
                    ok = mbar_wait_warp(bar(c_full, slot), turn_of(number, L::CODES)) && (is_v || mbar_wait_warp(bar(empty, my_stage), turn_of(number, L::STAGES) ^ 1u));
                    if (!ok) { failed(is_v ? 45 : 44); break; }
                    const uint32_t src = base + (is_v ? L::V_CODES : L::K_CODES) + slot * CODE_BYTES + half * 32 * D + lane * 16;
                    // this lane has the scale of a row: 2^fold, twice in a word, and what the fold leaves - as a factor of the key's score, or in log2
                    // units - which is read only where a flag says so, of either kind
                    const uint8_t* const scales = sh.code_scales[is_v][slot];
                    const int my_row = half * 32 + lane;
                    int scale0 = scales[0];
                    if (is_v) {                                                      // the largest, of the rows that every token sees; 1 where there are none
                        const int lo = key0 + lane < pos0 ? scales[lane] : 0, hi = key0 + 32 + lane < pos0 ? scales[32 + lane] : 0;
                        scale0 = key0 < pos0 ? __reduce_max_sync(0xffffffffu, max(lo, hi)) : Q3_SCALE_BIAS;
                    }
                    const int e = key0 + my_row < key_end ? (int)scales[my_row] - scale0 : 0;     // (the scale of a row that nobody wrote may be anything)
                    const int fold = min(max(e, FOLD_LOW), FOLD_HIGH);
                    const uint32_t by = (uint32_t)(fold + 15) * 0x04000400u;
                    uint32_t flags = e != fold ? 1u : 0u;
                    if (is_v) sh.value_rest[note][my_row] = (float)(e - fold);
                    else sh.key_rest[note][my_row] = q3_exp2i(e - fold);
                    if (edge && is_v) {
#pragma unroll 1
                        for (int i = 0; i < TURNS; ++i) {
                            const uint4 w = ld_shared_v4(src + i * AT_ONCE * D);
                            if (key0 + half * 32 + i * AT_ONCE + r_in < key_end && (no_numbers<true>(w.x) | no_numbers<true>(w.y) | no_numbers<true>(w.z) | no_numbers<true>(w.w)) != 0)
                                flags |= 2u;
                        }
                    }
                    flags = __reduce_or_sync(0xffffffffu, flags);
                    __syncwarp();
                    if (lane == 0) {
                        Note& to_note = is_v ? sh.values[note] : sh.keys[note];
                        to_note.flags[half] = flags;
                        if (half == 0) to_note.scale = is_v ? (float)(scale0 - Q3_SCALE_BIAS) : q3_exp2i(scale0 - Q3_SCALE_BIAS);
                        mbar_arrive(bar(L::NOTED, note));
                    }
                    if (is_v) {
                        ok = mbar_wait_warp(bar(empty, my_stage), turn_of(number, L::STAGES) ^ 1u);
                        if (!ok) { failed(36); break; }
                    }
                    // (few turns a round: the loops of all roles share an instruction cache; with twice as many everything took 1.05 times as long)
#pragma unroll 4
                    for (int i = 0; i < TURNS; ++i) {
                        uint32_t v[2][2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) load_words2(v[k], src + i * AT_ONCE * D + 8 * (k ^ swap));
                        if (edge && is_v) {
                            const bool live = key0 + half * 32 + i * AT_ONCE + r_in < key_end;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint32_t& w = v[k >> 1][k & 1];
                                w = live ? w & ~no_numbers<true>(w) : 0u;
                            }
                        }
                        const uint32_t mine = __shfl_sync(0xffffffffu, by, i * AT_ONCE + r_in);
                        const __half2 m = *reinterpret_cast<const __half2*>(&mine);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            uint32_t h[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const __half2 z = __hmul2(q3_half2_of(v[k][j >> 1] >> (16 * (j & 1))), m);
                                h[j] = *reinterpret_cast<const uint32_t*>(&z);
                            }
                            st_shared_v4((i & 1 ? to[1][k] : to[0][k]) + i * AT_ONCE * 128, make_uint4(h[0], h[1], h[2], h[3]));
                        }
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(bar(full, my_stage));
                        mbar_arrive(bar(c_empty, slot));
                    }
                }
            } else if (is_v) {
                // ------------------------------------------------ a look at the values of pages that some row does not see in whole
                for (int n = 0; n < steps; ++n) {
                    const int number = page0 + n, stage = number % L::STAGES, key0 = (part.begin + n) * PAGE;
                    ok = mbar_wait_warp(bar(L::V_HERE, stage), turn_of(number, L::STAGES));
                    if (!ok) { failed(46); break; }
                    if (key0 + PAGE > pos0) {
                        // values behind the end, and those that are no numbers, become zeros; a warp looks through 16 rows
                        uint32_t found = 0;
                        for (int i = lane; i < 16 * (D / 8); i += 32) {
                            const int row = w4 * 16 + i / (D / 8);
                            const uint32_t at_chunk = base + L::V + stage * TILE_BYTES + chunk_at(row, i % (D / 8), PANEL_BYTES);
                            uint4 v = ld_shared_v4(at_chunk);
                            const bool live = key0 + row < key_end;
                            if (!live) v = make_uint4(0, 0, 0, 0);
                            const uint4 bad = make_uint4(no_numbers<false>(v.x), no_numbers<false>(v.y), no_numbers<false>(v.z), no_numbers<false>(v.w));
                            const uint32_t any = bad.x | bad.y | bad.z | bad.w;
                            found |= any;
                            if (any != 0 || !live) st_shared_v4(at_chunk, make_uint4(v.x & ~bad.x, v.y & ~bad.y, v.z & ~bad.z, v.w & ~bad.w));
                        }
                        found = __reduce_or_sync(0xffffffffu, found);
                        if (lane == 0) sh.values[number % NOTES].flags[w4] = found != 0 ? 2u : 0u;
                        fence_proxy_async();
                        __syncwarp();
                    }
                    if (lane == 0) {
                        mbar_arrive(bar(L::V_FULL, stage));
                        mbar_arrive(bar(L::NOTED, number % NOTES));
                    }
                }
            }
            page0 += steps;
            at = Work::next(part);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MMA_REGS));
        if (warp == MMA_WARP || warp == MMA_WARP + 3) {
            // ------------------------------------------------ the products of a tile: the whole warp walks and one elected thread issues
            constexpr uint32_t idesc_s = idesc(F8, BM, PAGE, false), idesc_pv = idesc(F8, BM, D, true);
            const int x = warp == MMA_WARP ? 0 : 1;
            const uint32_t acc = __shfl_sync(0xffffffffu, tmem, 0) + x * TILE_COLS;
            const uint64_t q_desc = desc_k_major(base + L::QUERIES), k_desc = desc_k_major(base + L::K), v_desc = desc_mn_major(base + L::V, PANEL_BYTES);
            uint32_t q_turn = 0, count = 0;                                          // parity of the parts; this tile's pages so far
            // the stage of a page and its turn, counted along
            struct Place { uint32_t stage, turn; } k_at = {0, 0}, v_at = {0, 0};
            auto step_on = [](Place& at, int by) {
                at.stage += by;
                while (at.stage >= L::STAGES) {
                    at.stage -= L::STAGES;
                    at.turn ^= 1u;
                }
            };
            bool ok = true;
            for (int at = share.from; at < share.to && ok;) {
                const TreePart part = at == share.from ? sh.part : Work::part(st, share, at, blockIdx.x);
                if (part.begin >= part.end) break;
                const bool split = part.n_new * group - part.tile * ROWS <= BM;
                const int steps = part.end - part.begin, first = split ? x : 0, stride = split ? 2 : 1;
                auto scores = [&](uint32_t buffer) {                                 // of the page at k_at
                    if (!mbar_wait_warp(bar(L::K_FULL, k_at.stage), k_at.turn)) return false;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t q_src = q_desc + (uint64_t)((split ? 0 : x) * (Q_BYTES >> 4)), k_src = k_desc + (uint64_t)(k_at.stage * (TILE_BYTES >> 4));
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk)
                            tc_mma_ss(acc + COL_S + buffer * 64, q_src + (uint64_t)(((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4),
                                      k_src + (uint64_t)(((kk >> 2) * PANEL_BYTES + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
                        tc_commit(bar(L::S_FULL, 2 * x + buffer));
                        tc_commit(bar(L::K_EMPTY, k_at.stage));                      // (both tiles' have to be done, or this one's twice)
                        if (split) tc_commit(bar(L::K_EMPTY, k_at.stage));
                    }
                    __syncwarp();
                    step_on(k_at, stride);
                    return true;
                };
                Place k_next = k_at, v_next = v_at;                                  // behind this part
                step_on(k_next, steps % (2 * L::STAGES));
                step_on(v_next, steps % (2 * L::STAGES));
                step_on(k_at, first);
                step_on(v_at, first);
                if (lane == 0) mbar_arrive(bar(L::Q, 0));
                ok = mbar_wait_warp(bar(L::Q, 0), q_turn);
                q_turn ^= 1u;
                tc_fence_after();
                for (int b = 0; b < 2 && ok; ++b)
                    if (first + b * stride < steps) ok = scores((count + b) & 1u);
                if (!ok) { failed(47); break; }
                for (int n = first; n < steps; n += stride, ++count) {
                    const uint32_t buffer = count & 1u;
                    // what is there long before is waited for first
                    ok = mbar_wait_warp(bar(L::V_FULL, v_at.stage), v_at.turn) && mbar_wait_warp(bar(L::P_FULL, 2 * x + buffer), count >> 1 & 1u);
                    if (!ok) { failed(48); break; }
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t v_src = v_desc + (uint64_t)(v_at.stage * (TILE_BYTES >> 4));
#pragma unroll
                        for (int kk = 0; kk < PAGE / 16; ++kk)
                            tc_mma_ts(acc + COL_O, acc + COL_S + buffer * 64 + kk * 8, v_src + (uint64_t)((kk * 16 * 128) >> 4), idesc_pv, (n >= stride || kk > 0) ? 1u : 0u);
                        tc_commit(bar(L::PV_DONE, x));
                        tc_commit(bar(L::V_EMPTY, v_at.stage));
                        if (split) tc_commit(bar(L::V_EMPTY, v_at.stage));
                    }
                    __syncwarp();
                    step_on(v_at, stride);
                    if (n + 2 * stride < steps) {
                        // the scores of the page after the next go where these weights were, once the products with them are done
                        ok = mbar_wait_warp(bar(L::PV_DONE, x), count & 1u) && scores(buffer);
                        if (!ok) { failed(51); break; }
                    }
                }
                k_at = k_next;
                v_at = v_next;
                at = Work::next(part);
            }
        } else if (warp == K_COPY_WARP || warp == V_COPY_WARP) {
            // ------------------------------------------------ copies of the keys, of the values
            const bool is_v = warp == V_COPY_WARP;
            int number = 0;
            bool ok = true;
            for (int at = share.from; at < share.to && ok;) {
                const TreePart part = at == share.from ? sh.part : Work::part(st, share, at, blockIdx.x);
                if (part.begin >= part.end) break;
                const int* table = st.page_table + (int64_t)part.seq * st.pages_per_seq;
                int64_t page = page_of(st, table, part.begin);
                for (int i = part.begin; i < part.end; ++i, ++number) {
                    const int64_t cell = (page * st.nkv + part.head) * PAGE;
                    if (i + 1 < part.end) page = page_of(st, table, i + 1);
                    if constexpr (F8) {
                        const int slot = number % L::CODES;
                        ok = mbar_wait_warp(bar(is_v ? L::VC_EMPTY : L::KC_EMPTY, slot), turn_of(number, L::CODES) ^ 1u);
                        if (!ok) { failed(is_v ? 50 : 49); break; }
                        if (lane == 0) {
                            const uint32_t full = bar(is_v ? L::VC_FULL : L::KC_FULL, slot);
                            mbar_expect_tx(full, CODE_BYTES + PAGE);
                            copy_bulk(base + (is_v ? L::V_CODES : L::K_CODES) + slot * CODE_BYTES, (is_v ? a.values : a.keys) + cell * D, CODE_BYTES, full);
                            copy_bulk(smem_u32(sh.code_scales[is_v][slot]), (is_v ? a.value_scales : a.key_scales) + cell, PAGE, full);
                        }
                    } else {
                        const int stage = number % L::STAGES;
                        ok = mbar_wait_warp(bar(is_v ? L::V_EMPTY : L::K_EMPTY, stage), turn_of(number, L::STAGES) ^ 1u);
                        if (!ok) { failed(is_v ? 50 : 49); break; }
                        if (lane == 0) {
                            const uint32_t full = bar(is_v ? L::V_HERE : L::K_FULL, stage), dst = base + (is_v ? L::V : L::K) + stage * TILE_BYTES;
                            mbar_expect_tx(full, TILE_BYTES);
#pragma unroll
                            for (int h = 0; h < HALVES; ++h) tma_load_2d(dst + h * PANEL_BYTES, is_v ? &map_v : &map_k, full, h * 64, (int)cell);
                        }
                    }
                    __syncwarp();
                }
                at = Work::next(part);
            }
            // its last copies have landed before the block goes, also where another role has given up
            constexpr int RING = F8 ? L::CODES : L::STAGES;
            for (int i = max(0, number - RING); i < number; ++i)
                mbar_wait_warp(bar(F8 ? (is_v ? L::VC_FULL : L::KC_FULL) : is_v ? L::V_HERE : L::K_FULL, i % RING), turn_of(i, RING));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// ---- the parts of the items that several blocks share, added up in their order: for every block of the first kernel that noted one, and for 32 of its rows, a block
constexpr int MERGE_THREADS = D / 8 * 32;
__global__ void __launch_bounds__(MERGE_THREADS) tree_tc_merge_kernel(const __grid_constant__ Args a, int blocks) {
    pdl_launch_dependents();
    pdl_wait();
    const int4* note = reinterpret_cast<const int4*>(a.parts + (int64_t)2 * blocks * PART) + 2 * blockIdx.x;
    const int4 n0 = note[0], n1 = note[1];
    const int parts = n0.x, slot0 = n0.y, first_block = n0.z, rows = n0.w, r = blockIdx.y * 32 + (threadIdx.x & 31);
    if (parts == 0 || r >= rows) return;
    const int group = a.step.nq / a.step.nkv, row = n1.x + r;
    bf16* const out = a.out + ((int64_t)(n1.y + row / group) * a.step.nq + n1.z * group + row % group) * D;
    const int c = threadIdx.x >> 5;                                                  // eight values a warp
    float m = -INFINITY, l = 0.0f, v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    constexpr int AT_ONCE = 4;                                                       // parts asked for together
    for (int b0 = 0; b0 < parts; b0 += AT_ONCE) {
        float2 ml[AT_ONCE];
        float4 u[AT_ONCE][2];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            const int i = min(b0 + k, parts - 1);
            const float* src = a.parts + (int64_t)(i == 0 ? slot0 : 2 * (first_block + i)) * PART;
            ml[k] = *reinterpret_cast<const float2*>(src + ROWS * D + 2 * r);
            u[k][0] = *reinterpret_cast<const float4*>(src + ((2 * c) * ROWS + r) * 4);
            u[k][1] = *reinterpret_cast<const float4*>(src + ((2 * c + 1) * ROWS + r) * 4);
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
            if (b0 + k >= parts) break;
            const float m2 = fmaxf(m, ml[k].x), was = m == m2 ? 1.0f : ex2(m - m2), now = ml[k].x == m2 ? 1.0f : ex2(ml[k].x - m2);
            m = m2;
            l = fmaf(now, ml[k].y, l * was);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = fmaf(now, (&u[k][0].x)[e], v[e] * was);
                v[e + 4] = fmaf(now, (&u[k][1].x)[e], v[e + 4] * was);
            }
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

template <bool F8> int launch(const Args& a, int max_new, cudaStream_t stream) {
    static Q3PerDevice configured;
    const cudaError_t e = q3_allow_shared_memory(tree_tc_kernel<F8>, smem_bytes<F8>, configured);
    if (e != cudaSuccess) return (int)e;
    CUtensorMap map_k = {}, map_v = {};
    if (!F8 && (!q3_make_map_bf16(&map_k, a.keys, a.step.n_pages * a.step.nkv * PAGE, D, PAGE, 64, true) ||
                !q3_make_map_bf16(&map_v, a.values, a.step.n_pages * a.step.nkv * PAGE, D, PAGE, 64, true)))
        return Q3_ERR_BAD_SIZE;
    const int64_t units = Work::most_units(a.step, PART_PAGES);
    if (units > 0x3fffffff) return Q3_ERR_TOO_LARGE;
    const int64_t most = (Work::most_units(a.step, 0) + LEAST_PAGES - 1) / LEAST_PAGES + Work::most_items(a.step);
    const int sms = q3_device_sm_count(), blocks = (int)(most < sms ? most : sms);
    int code = (int)q3_launch(tree_tc_kernel<F8>, dim3(blocks), dim3(THREADS), (size_t)smem_bytes<F8>, stream, map_k, map_v, a);
    if (code != 0) return code;
    const int rows = (int64_t)max_new * (a.step.nq / a.step.nkv) < ROWS ? max_new * (a.step.nq / a.step.nkv) : ROWS;
    return (int)q3_launch(tree_tc_merge_kernel, dim3(blocks, (rows + 31) / 32), dim3(MERGE_THREADS), 0, stream, a, blocks);
}

}  // namespace

Q3_EXPORT int q3_attention_tree_tc_head_dim() { return D; }

// Float32 values of `parts` for a launch.
Q3_EXPORT int64_t q3_attention_tree_tc_parts() { return q3_device_sm_count() * ((int64_t)2 * PART + sizeof(MergeNote) / sizeof(float)); }

Q3_EXPORT int q3_attention_tree_tc_bf16(const q3_attention_tree_args* x) {
    if (x->n_seqs <= 0 || x->max_new <= 0) return 0;
    const int refused = tree_refused(*x, D);
    if (refused != 0) return refused;
    if (!(x->scale > 0.0)) return Q3_ERR_BAD_SIZE;                                   // the maximum is taken before the scale
    if (x->n_pages * x->nkv * PAGE > 0x7fffffff) return Q3_ERR_TOO_LARGE;            // a row's number is a coordinate of a copy
    const Args a = {tree_step(*x), (const bf16*)x->q, (bf16*)x->out, (const unsigned char*)x->k_pages, (const unsigned char*)x->v_pages,
                    (const uint8_t*)x->k_scales, (const uint8_t*)x->v_scales, (float*)x->parts, (int*)x->status, (float)x->scale * 1.4426950408889634f};
    return x->k_scales != nullptr ? launch<true>(a, x->max_new, (cudaStream_t)x->stream) : launch<false>(a, x->max_new, (cudaStream_t)x->stream);
}
