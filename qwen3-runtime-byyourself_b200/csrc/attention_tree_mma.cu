// Attention of a step's new tokens - one, a run or a tree of drafted ones a sequence - over the cache's pages in bfloat16 or in 8 bits, for
// few rows (a row: a token and query head) a kv head: 8, 16 or 32 at a time.  What a token sees and what comes out is said in attention_tree.cu.
//
// Few rows read many keys, so the floor is the time of the cached rows from memory: 2 (d + 1) bytes a token and kv head in 8 bits.
//   - A block of four warps takes an equal share of the pages of all (sequence, kv head, tile of rows) (tree_work.cuh), three blocks an SM.
//   - A warp takes every fourth step of 32 (16) keys of its block's, by itself: it copies the step's keys and values into shared memory with
//     asynchronous copies a step or two ahead, laid so that a lane reads runs of 16 bytes without bank conflicts; no barrier is met.
//   - Products are mma.m16n8k16 with keys, then values, as the 16-row operand and the rows as its eight columns: S^T = K Q^T and O^T = V^T P^T, so 8 rows
//     cost 8, not 16.  What a lane holds of keys and values are runs of 16 bytes, which fixes the order in which the products walk a
//     head's values and the keys; the query is read in the same order.  The weights change from rows to columns by movmatrix.
//   - 8 bits: a code is exact in half precision and becomes that in one conversion a pair (products of the codes themselves were tried and gained
//     nothing).  Queries are divided by a power of two for each row, so that they fit, exactly, unless a value is below 2^-24 of its
//     row's largest.  The key's scale multiplies the score.  The value's scale 2^v is part of the weight: w = 2^(x + v - M), x the score in log2 units
//     and M the running maximum of x + v, so the largest weight is of the order of 1 whatever the scales are, and what half precision drops is
//     below 2^-24 of the largest term; the sum of the softmax is that of w 2^-v, in 32 bits.
//   - The maximum is raised only when it is exceeded by more than 2^8.
//   - One new token, 32 heads over 8 (8 bits): 64 sequences of up to 9,000 keys (40 heads) 109 us, 5.6 TB/s of the 6.5 that a copy reaches; 8 of up to 4,000
//     17.9 (the floor is 6.6: of 23,000 cycles 3,000 go by until a block knows its share, 3,500 until its copies are under way, 9,000 for its six pages, 1,500 until
//     its warps' sums have met and 5,000 until the parts of a row have), one of 32,000 26.8, one of 130 7.4.
//   - A step with new tokens masks by bits; a value that is no number reaches only the rows that see it (a product of 0 and a NaN is a NaN:
//     such values are taken out before the product and added to the rows that see them).
#include "page8.cuh"
#include "tree_work.cuh"

#ifndef Q3_HEAD_DIM
#error "compile with -DQ3_HEAD_DIM=<64 or 128>"
#endif

namespace {

constexpr int D = Q3_HEAD_DIM, PAGE = Q3_PAGE_TOKENS;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
static_assert(PAGE == 64, "a page holds 64 tokens");
constexpr int WARPS = 4;
// Blocks an SM and stages of a warp's ring, by tiles of eight rows (registers, shared memory).
template <int NT> constexpr int blocks_per_sm = NT == 4 ? 2 : 3;
template <int NT> constexpr int stages = NT == 4 ? 3 : 2;
// A block is given no fewer pages, and all of items of up to WHOLE_PAGES (130 keys whole 7.4 us, in two parts 8.2; 600 whole 11.0, in five 9.1); in the time of
// how many pages a part is added up, for every 128 packets of its rows: 0 (and four pages at least) / 0.1 / 0.2 / 0.3 for 1 sequence of 32,000 keys of 2 kv heads, 4
// tokens and 8 heads 65 / 34 / 32 / 34 us, 3 of up to 30,000 of one, 1 and 8 (bfloat16) 31 / 24 / 24 / 25, 1 of 8,000 of 4, 2 and 16 16.1 / 16.2 / 17.3 / 18.6.
constexpr int LEAST_PAGES = 2, WHOLE_PAGES = 4;
constexpr float JOIN_PAGES = 0.2f;
// Pages that take about as long as beginning and ending a part.  0 / 4 / 8 / 12: 64 sequences of up to 2,000 keys and one new token (8 bits) 57 / 44 / 42 / 42 us,
// of up to 9,000 123 / 113 / 113 / 110, with four new tokens 129 / 102 / 83 / 82, of 130 20 / 14.6 / 15.2 / 15.2.
constexpr int PART_PAGES = 8;
constexpr float RAISE = 8.0f;

template <bool F8> struct Form {
    static constexpr int KEYS = F8 || D == 64 ? 32 : 16;              // keys of a step
    static constexpr int TILES = KEYS / 16, MINE = KEYS / 8, OWN = KEYS / 4;   // tiles of 16 keys; keys and values of a step that a lane holds
    static constexpr int ROW = D * (F8 ? 1 : 2);                      // bytes of a cached row
    static constexpr int K_RUNS = ROW / 64;                           // 16-byte runs of a key a lane holds
    static constexpr int V_BYTES = ROW / 8;                           // bytes of a value a lane holds: in runs of V_RUN
    static constexpr int V_RUN = V_BYTES < 16 ? V_BYTES : 16, V_RUNS = V_BYTES / V_RUN;
    static constexpr int SPAN = V_RUN / (F8 ? 1 : 2);                 // values of a run: lanes g hold values g SPAN .. of a group of 8 SPAN
    // Where the run of lane (g, t) lies among 32: a row's runs side by side, which is how eight lanes copy them (four rows' runs of a lane's neighbours are
    // half sectors: 24 sectors a copy instead of 16), turned so that lanes that read together do not meet in a bank.
    static __device__ __forceinline__ uint32_t value_at(int g, int t) { return (t * 8 + (g ^ (V_RUN == 16 ? 2 * t : 4 * (t >> 1)))) * V_RUN; }
    static constexpr int K_BYTES = MINE * K_RUNS * 512, STAGE = K_BYTES + OWN * V_RUNS * 32 * V_RUN;
};

constexpr int Q_PITCH = D * 2 + 8;
template <bool F8, int NT> constexpr int smem_ring = WARPS * stages<NT> * Form<F8>::STAGE;
template <int NT> constexpr int merge_bytes = WARPS * 8 * NT * D * 4;
template <bool F8, int NT> constexpr int area = smem_ring<F8, NT> > merge_bytes<NT> ? smem_ring<F8, NT> : merge_bytes<NT>;
template <bool F8, int NT> constexpr int smem_bytes =
    area<F8, NT> + WARPS * stages<NT> * 64 + 8 * NT * Q_PITCH + 8 * NT * 4 + 2 * WARPS * 8 * NT * 4 + 64;

struct Args {
    TreeStep step;
    const bf16* q;
    bf16* out;
    const unsigned char *keys, *values;
    const uint8_t *key_scales, *value_scales;
    float* parts;
    int* counters;
    float scale_log2;
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int N> __device__ __forceinline__ void load_words(uint32_t* w, uint32_t at) {
    if constexpr (N == 16) asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    else asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
}

template <bool F8> __device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (F8)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// An 8 x 8 tile of 16-bit values, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool F8> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (F8) {
        const __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}
__device__ __forceinline__ uint32_t half2_bits(uint32_t codes) {
    const __half2 v = q3_half2_of(codes);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The values of a word that are infinities or NaNs, each marked by all of its bits.
template <bool F8> __device__ __forceinline__ uint32_t no_numbers(uint32_t w) {
    if constexpr (F8) return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
    else return ((((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
}

// Where the float4 number f of a row lies in the buffer in which the warps' sums meet: lanes that write together do not meet in a bank.
template <int SPAN> __device__ __forceinline__ int meet_at(int row, int f) {
    if constexpr (SPAN == 16) return f ^ (row >> 1 & 3);
    else return f ^ ((row >> 1 & 1) | (row >> 2 & 1) << 2);
}

template <bool F8, int NT>
__global__ void __launch_bounds__(WARPS * 32, blocks_per_sm<NT>) tree_mma_kernel(const __grid_constant__ Args a) {
    using F = Form<F8>;
    constexpr int ROWS = 8 * NT, KEYS = F::KEYS, TILES = F::TILES, OWN = F::OWN, MINE = F::MINE, M_TILES = D / 16, K_STEPS = D / 16;
    constexpr int PART = ROWS * (D + 2), STAGES = stages<NT>;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char* const q_rows = smem + area<F8, NT> + WARPS * STAGES * 64;
    float* const row_factor = reinterpret_cast<float*>(q_rows + ROWS * Q_PITCH);
    float* const warp_max = row_factor + ROWS;                        // [WARPS][ROWS]
    float* const warp_sum_of = warp_max + WARPS * ROWS;
    TreeShare* const shared_share = reinterpret_cast<TreeShare*>(warp_sum_of + WARPS * ROWS);
    int* const shared_last = reinterpret_cast<int*>(shared_share + 1);
    pdl_launch_dependents();
    pdl_wait();
    const TreeStep& st = a.step;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    using Work = TreeWork<PAGE, ROWS, false>;
    const int group = st.nq / st.nkv;

    if (warp == 0) {
        const int most_rows = (int)min((int64_t)ROWS, (int64_t)st.max_new * group);
        const float join = JOIN_PAGES * (float)((most_rows * (D / 4) + WARPS * 32 - 1) / (WARPS * 32));
        const TreeShare found = Work::share(st, LEAST_PAGES, WHOLE_PAGES, join, PART_PAGES, blockIdx.x, gridDim.x);
        if (lane == 0) *shared_share = found;
    }
    __syncthreads();
    TreeShare share = *shared_share;

    const uint32_t ring = smem_at(smem) + warp * (STAGES * F::STAGE), scales = smem_at(smem) + area<F8, NT> + warp * (STAGES * 64);

    for (int at = share.from; at < share.to;) {
        const TreePart part = Work::part(st, share, at, blockIdx.x);
        if (part.begin >= part.end) break;
        const int t0 = part.t0, n_new = part.n_new, pos0 = part.pos0;
        const int row0 = part.tile * ROWS, rows = min(ROWS, n_new * group - row0);      // row i of the tile: token (row0 + i) / group, head (row0 + i) % group
        const int key_begin = part.begin * PAGE, key_end = min(part.end * PAGE, pos0 + n_new);
        const int steps = (key_end - key_begin + KEYS - 1) / KEYS;
        const int* table = st.page_table + (int64_t)part.seq * st.pages_per_seq;

        // ---- copies of a step's rows; the page of the step after it is asked for meanwhile
        auto page_of = [&](int s) {
            if (s >= steps) return 0;
            const int p = table[(key_begin + s * KEYS) / PAGE];
            return p >= 0 && p < st.n_pages ? p : 0;                 // (a number that is no page: stay within the cache)
        };
        int next_page = page_of(warp);
        // the warp's rows of queries are asked for before the copies, which wait for the page table
        constexpr int PER = D / 32, MY_ROWS = ROWS / WARPS;
        uint32_t q_raw[MY_ROWS][PER / 2];
#pragma unroll
        for (int i = 0; i < MY_ROWS; ++i) {
            const int r = warp + i * WARPS;
            const bf16* src = a.q + ((int64_t)(t0 + (row0 + min(r, rows - 1)) / group) * st.nq + part.head * group + (row0 + min(r, rows - 1)) % group) * D + lane * PER;
#pragma unroll
            for (int e = 0; e < PER / 2; ++e) q_raw[i][e] = r < rows ? reinterpret_cast<const uint32_t*>(src)[e] : 0u;
        }
        auto issue = [&](int s, int stage) {
            if (s < steps) {
                const int64_t cell0 = ((int64_t)next_page * st.nkv + part.head) * PAGE + ((key_begin + s * KEYS) & (PAGE - 1));
                next_page = page_of(s + WARPS);
                const unsigned char *k = a.keys + cell0 * F::ROW, *v = a.values + cell0 * F::ROW;
                const uint32_t dst = ring + stage * F::STAGE;
#pragma unroll
                for (int j = 0; j < MINE; ++j)
#pragma unroll
                    for (int h = 0; h < F::K_RUNS; ++h)
                        copy_async<16>(dst + (j * F::K_RUNS + h) * 512 + lane * 16, k + (MINE * g + j) * F::ROW + h * 64 + t * 16);
#pragma unroll
                for (int i = 0; i < OWN; ++i)
#pragma unroll
                    for (int h = 0; h < F::V_RUNS; ++h)
                        copy_async<F::V_RUN>(dst + F::K_BYTES + (i * F::V_RUNS + h) * 32 * F::V_RUN + F::value_at(lane & 7, lane >> 3),
                                             v + (OWN * (lane >> 3) + i) * F::ROW + h * 128 + (lane & 7) * F::V_RUN);
                if constexpr (F8) {
                    if (lane < 16) copy_async<4>(scales + stage * 64 + lane * 4, (lane < 8 ? a.key_scales : a.value_scales) + cell0 + (lane & 7) * 4);
                }
            }
            copy_commit();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) issue(warp + i * WARPS, i);

        // ---- the tile's queries, in half precision behind a power of two a row, or as they are
#pragma unroll
        for (int i = 0; i < MY_ROWS; ++i) {
            const int r = warp + i * WARPS;
            const bf16* x = reinterpret_cast<const bf16*>(q_raw[i]);
            uint32_t* dst = reinterpret_cast<uint32_t*>(q_rows + r * Q_PITCH + lane * PER * 2);
            if constexpr (F8) {
                float top = 0.0f;
#pragma unroll
                for (int e = 0; e < PER; ++e) top = fmaxf(top, fabsf(__bfloat162float(x[e])));
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                int e2 = (int)(__float_as_uint(top) >> 23) - 127;
                e2 = e2 >= 128 ? 0 : min(max(e2, -60), 60);
                const float down = q3_exp2i(-e2);
#pragma unroll
                for (int e = 0; e < PER; e += 2) dst[e / 2] = pack2<true>(__bfloat162float(x[e]) * down, __bfloat162float(x[e + 1]) * down);
                if (lane == 0) row_factor[r] = a.scale_log2 * q3_exp2i(e2);
            } else {
#pragma unroll
                for (int e = 0; e < PER / 2; ++e) dst[e] = q_raw[i][e];
            }
        }
        __syncthreads();

        // the columns' operand of product ks: 16 of a head's values, in the order in which a lane holds keys
        const uint32_t q_at = smem_at(q_rows) + g * Q_PITCH + (F8 ? 32 : 16) * t;
        auto load_q = [&](int n, int ks, uint32_t* f) {
            load_words<8>(f, q_at + n * 8 * Q_PITCH + (F8 ? (ks >> 2) * 128 + (ks & 3) * 8 : (ks >> 1) * 64 + (ks & 1) * 8));
        };
        constexpr bool KEEP_Q = NT <= 2;
        uint32_t q_frag[KEEP_Q ? NT : 1][KEEP_Q ? K_STEPS : 1][2];
        if constexpr (KEEP_Q) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int ks = 0; ks < K_STEPS; ++ks) load_q(n, ks, q_frag[n][ks]);
        }
        float factor[NT][2];
        int own[NT][2];                                              // the token of a column's row, among the sequence's new ones
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int row = n * 8 + 2 * t + b;
                factor[n][b] = F8 ? row_factor[row] : a.scale_log2;
                own[n][b] = (row0 + min(row, rows - 1)) / group;
            }

        float o[NT][M_TILES][4], m_run[NT][2], l_run[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < M_TILES; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
            m_run[n][0] = m_run[n][1] = -INFINITY;
            l_run[n][0] = l_run[n][1] = 0.0f;
        }

        int stage = 0;
        for (int s = warp; s < steps; s += WARPS) {
            issue(s + (STAGES - 1) * WARPS, stage == 0 ? STAGES - 1 : stage - 1);
            copy_wait<STAGES - 1>();
            __syncwarp();
            const uint32_t here = ring + stage * F::STAGE;
            const int key0 = key_begin + s * KEYS;
            const bool edge = key0 + KEYS > pos0;                    // some key of the step is a new token's, or behind the end

            // ---- scores: this lane's are those of keys MINE g .. + MINE - 1 and columns 2 t, 2 t + 1 of every tile
            float sc[NT][TILES][4];                                  // [key 2 j][column 0, 1], [key 2 j + 1][column 0, 1]
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < TILES; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[n][j][e] = 0.0f;
#pragma unroll
            for (int h = 0; h < F::K_RUNS; ++h) {
                constexpr int INNER = F8 ? 4 : 2;                    // products of a run
                uint32_t w[MINE][4];
#pragma unroll
                for (int j = 0; j < MINE; ++j) load_words<16>(w[j], here + (j * F::K_RUNS + h) * 512 + lane * 16);
#pragma unroll
                for (int m = 0; m < INNER; ++m) {
                    uint32_t k[TILES][4];
#pragma unroll
                    for (int j = 0; j < TILES; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t* run = w[2 * j + e];
                            k[j][e] = F8 ? half2_bits(run[m]) : run[2 * (m & 1)];
                            k[j][2 + e] = F8 ? half2_bits(run[m] >> 16) : run[2 * (m & 1) + 1];
                        }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        uint32_t f[2];
                        const uint32_t* q = f;
                        if constexpr (KEEP_Q) q = q_frag[n][h * INNER + m];
                        else load_q(n, h * INNER + m, f);
#pragma unroll
                        for (int j = 0; j < TILES; ++j) mma<F8>(sc[n][j], k[j], q[0], q[1]);
                    }
                }
            }

            // ---- in log2 units, with the scales of keys and values; what is not seen is minus infinity
            float back[MINE];                                        // 2^-v
            if constexpr (F8) {
                uint32_t kw, vw;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(kw) : "r"(scales + stage * 64 + g * MINE) : "memory");
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(vw) : "r"(scales + stage * 64 + 32 + g * MINE) : "memory");
#pragma unroll
                for (int i = 0; i < MINE; ++i) {
                    const uint32_t kb = (kw >> (8 * i)) & 0xffu, vb = (vw >> (8 * i)) & 0xffu;
                    const float ks = __uint_as_float(kb << 23), v = __uint_as_float(0x4b000000u | vb) - (8388608.0f + Q3_SCALE_BIAS);
                    back[i] = __uint_as_float(0x7f000000u - (vb << 23));
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            float& x = sc[n][i >> 1][2 * (i & 1) + b];
                            x = fmaf(x * ks, factor[n][b], v);
                        }
                }
            } else {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < TILES; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[n][j][e] *= a.scale_log2;
            }
            uint32_t seen[NT][2];                                    // of the step's keys, by row
            if (edge) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const unsigned long long* mask = st.tree != nullptr ? st.tree + (int64_t)(t0 + own[n][b]) * st.words : nullptr;
                        seen[n][b] = (uint32_t)tree_seen(mask, st.words, pos0, n_new, own[n][b], key0);
#pragma unroll
                        for (int i = 0; i < MINE; ++i)
                            if (!(seen[n][b] >> (MINE * g + i) & 1u)) sc[n][i >> 1][2 * (i & 1) + b] = -INFINITY;
                    }
                if constexpr (F8) {                                  // (the scale of a row that nobody wrote may be anything)
#pragma unroll
                    for (int i = 0; i < MINE; ++i)
                        if (key0 + MINE * g + i >= pos0 + n_new) back[i] = 0.0f;
                }
            }

            // ---- the running maximum
            float top[NT][2];
            bool raise = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float x = fmaxf(sc[n][0][b], sc[n][0][2 + b]);
#pragma unroll
                    for (int j = 1; j < TILES; ++j) x = fmaxf(x, fmaxf(sc[n][j][b], sc[n][j][2 + b]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    top[n][b] = x;
                    raise |= x > m_run[n][b] + RAISE;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        if (top[n][b] > m_run[n][b]) {
                            const float alpha = ex2(m_run[n][b] - top[n][b]);
                            m_run[n][b] = top[n][b];
                            l_run[n][b] *= alpha;
#pragma unroll
                            for (int i = 0; i < M_TILES; ++i) {
                                o[n][i][b] *= alpha;
                                o[n][i][2 + b] *= alpha;
                            }
                        }
                    }
            }

            // ---- weights, as the columns' operand
            uint32_t p[NT][TILES][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float m0 = m_run[n][0] == -INFINITY ? 0.0f : m_run[n][0], m1 = m_run[n][1] == -INFINITY ? 0.0f : m_run[n][1];      // nothing seen so far
#pragma unroll
                for (int j = 0; j < TILES; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = ex2(sc[n][j][2 * e] - m0), y = ex2(sc[n][j][2 * e + 1] - m1);
                        l_run[n][0] = F8 ? fmaf(x, back[2 * j + e], l_run[n][0]) : l_run[n][0] + x;
                        l_run[n][1] = F8 ? fmaf(y, back[2 * j + e], l_run[n][1]) : l_run[n][1] + y;
                        p[n][j][e] = transposed(pack2<F8>(x, y));
                    }
            }

            // ---- weighted values: tile j's products walk keys OWN t + {2 j, OWN / 2 + 2 j, 2 j + 1, OWN / 2 + 2 j + 1} of every lane
            uint32_t odd = 0;                                        // some value of the step is no number
#pragma unroll
            for (int j = 0; j < TILES; ++j)
#pragma unroll
                for (int h = 0; h < F::V_RUNS; ++h) {
                    constexpr int W = F::V_RUN / 4;
                    uint32_t w[4][W];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = (i & 1) * (OWN / 2) + 2 * j + (i >> 1);
                        load_words<F::V_RUN>(w[i], here + F::K_BYTES + (key * F::V_RUNS + h) * 32 * F::V_RUN + F::value_at(g, t));
                        if (edge) {
                            const bool dead = key0 + OWN * t + key >= pos0 + n_new;
#pragma unroll
                            for (int k = 0; k < W; ++k) {
                                if (dead) w[i][k] = 0u;
                                const uint32_t bad = no_numbers<F8>(w[i][k]);
                                odd |= bad;
                                w[i][k] &= ~bad;
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < W; ++k) {
                        if constexpr (F8) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t x = __byte_perm(w[0][k], w[1][k], e ? 0x7362 : 0x5140), y = __byte_perm(w[2][k], w[3][k], e ? 0x7362 : 0x5140);
                                const uint32_t v[4] = {half2_bits(x), half2_bits(x >> 16), half2_bits(y), half2_bits(y >> 16)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma<true>(o[n][(h * F::SPAN + 4 * k) / 2 + e], v, p[n][j][0], p[n][j][1]);
                            }
                        } else {
                            const uint32_t v[4] = {__byte_perm(w[0][k], w[1][k], 0x5410), __byte_perm(w[0][k], w[1][k], 0x7632),
                                                   __byte_perm(w[2][k], w[3][k], 0x5410), __byte_perm(w[2][k], w[3][k], 0x7632)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma<false>(o[n][(h * F::SPAN + 2 * k) / 2], v, p[n][j][0], p[n][j][1]);
                        }
                    }
                }
            if (edge && __any_sync(0xffffffffu, odd != 0)) {
                // the values that are no numbers, to the rows that see their keys
#pragma unroll 1
                for (int key = 0; key < KEYS; ++key) {
                    if (key0 + key >= pos0 + n_new) break;
                    const uint32_t src = here + F::K_BYTES;
#pragma unroll
                    for (int h = 0; h < F::V_RUNS; ++h) {
                        uint32_t w[F::V_RUN / 4];
                        load_words<F::V_RUN>(w, src + ((key % OWN) * F::V_RUNS + h) * 32 * F::V_RUN + F::value_at(g, key / OWN));
#pragma unroll
                        for (int e = 0; e < F::SPAN; ++e) {
                            float v;
                            uint32_t bad;
                            if constexpr (F8) {
                                bad = no_numbers<true>(w[e / 4]) >> (8 * (e & 3)) & 1u;
                                v = __uint_as_float(0x7fffffffu);
                            } else {
                                bad = no_numbers<false>(w[e / 2]) >> (16 * (e & 1)) & 1u;
                                v = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int b = 0; b < 2; ++b)
                                    if (bad && (seen[n][b] >> key & 1u)) o[n][(h * F::SPAN + e) / 2][2 * (e & 1) + b] += v;
                        }
                    }
                }
            }
            __syncwarp();                                            // the stage is read: it may be copied over
            stage = stage + 1 == STAGES ? 0 : stage + 1;
        }
        copy_wait<0>();
        __syncthreads();                                             // every warp is done with the ring

        // ---- the warps' sums meet
        float* const meet = reinterpret_cast<float*>(smem);
        const bool some = warp < steps;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int row = n * 8 + 2 * t + b;
                float l = l_run[n][b];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) {
                    warp_max[warp * ROWS + row] = m_run[n][b];
                    warp_sum_of[warp * ROWS + row] = l;
                }
                if (some && row < rows) {
#pragma unroll
                    for (int h = 0; h < F::V_RUNS; ++h)
#pragma unroll
                        for (int q = 0; q < F::SPAN / 4; ++q) {
                            const int f = (h * 64 + g * F::SPAN) / 4 + q, i = (h * F::SPAN + 4 * q) / 2;
                            reinterpret_cast<float4*>(meet)[(warp * ROWS + row) * (D / 4) + meet_at<F::SPAN>(row, f)] =
                                make_float4(o[n][i][b], o[n][i][2 + b], o[n][i + 1][b], o[n][i + 1][2 + b]);
                        }
                }
            }
        __syncthreads();
        const bool whole = part.parts == 1;
        const int met = min(WARPS, steps);
        auto place = [&](int row, int f) { return a.out + ((int64_t)(t0 + (row0 + row) / group) * st.nq + part.head * group + (row0 + row) % group) * D + 4 * f; };
        auto put = [&](int row, int f, float4 v, float l) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint2 w;
            w.x = pack2<false>(v.x * inv, v.y * inv);
            w.y = pack2<false>(v.z * inv, v.w * inv);
            *reinterpret_cast<uint2*>(place(row, f)) = w;
        };
        for (int i = threadIdx.x; i < rows * (D / 4); i += WARPS * 32) {
            const int row = i / (D / 4), f = i % (D / 4);
            float m = -INFINITY, l = 0.0f;
            for (int w = 0; w < met; ++w) m = fmaxf(m, warp_max[w * ROWS + row]);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int w = 0; w < met; ++w) {
                const float mw = warp_max[w * ROWS + row], alpha = mw == m ? 1.0f : ex2(mw - m);
                const float4 u = reinterpret_cast<const float4*>(meet)[(w * ROWS + row) * (D / 4) + meet_at<F::SPAN>(row, f)];
                l = fmaf(alpha, warp_sum_of[w * ROWS + row], l);
                v.x = fmaf(alpha, u.x, v.x); v.y = fmaf(alpha, u.y, v.y); v.z = fmaf(alpha, u.z, v.z); v.w = fmaf(alpha, u.w, v.w);
            }
            if (whole) {
                put(row, f, v, l);
            } else {
                float* dst = a.parts + (int64_t)part.slot * PART;
                *reinterpret_cast<float4*>(dst + row * D + 4 * f) = v;
                if (f == 0) *reinterpret_cast<float2*>(dst + ROWS * D + 2 * row) = make_float2(m, l);
            }
        }
        if (!whole) {
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();                                     // (of the block's writes, which the barrier has put before it)
                *shared_last = atomicAdd(a.counters + part.item, 1) == part.parts - 1 ? 1 : 0;
                if (*shared_last) a.counters[part.item] = 0;
                __threadfence();
            }
            __syncthreads();
            if (*shared_last) {
                for (int i = threadIdx.x; i < rows * (D / 4); i += WARPS * 32) {
                    const int row = i / (D / 4), f = i % (D / 4);
                    float m = -INFINITY, l = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    auto add = [&](int b) {
                        const float* src = a.parts + (int64_t)part.slot_of(b) * PART;
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + ROWS * D + 2 * row));
                        const float4 u = __ldcg(reinterpret_cast<const float4*>(src + row * D + 4 * f));
                        const float m2 = fmaxf(m, ml.x), was = m == m2 ? 1.0f : ex2(m - m2), now = ml.x == m2 ? 1.0f : ex2(ml.x - m2);
                        m = m2;
                        l = fmaf(now, ml.y, l * was);
                        v.x = fmaf(now, u.x, v.x * was); v.y = fmaf(now, u.y, v.y * was);
                        v.z = fmaf(now, u.z, v.z * was); v.w = fmaf(now, u.w, v.w * was);
                    };
                    int b = 0;
                    // (eight at once where there are many: one token of 32 heads over 32,000 keys has 51, 28.3 -> 26.3 us)
                    if constexpr (NT == 1)
#pragma unroll 1
                        for (; b + 16 <= part.parts; b += 8)
#pragma unroll
                            for (int k = 0; k < 8; ++k) add(b + k);
#pragma unroll 4
                    for (; b < part.parts; ++b) add(b);
                    put(row, f, v, l);
                }
            }
        }
        __syncthreads();                                             // the buffers are free for the next part
        at = Work::next(part);
    }
}

template <bool F8, int NT> int launch(const Args& a, int sm_count, cudaStream_t stream) {
    static Q3PerDevice configured;
    constexpr int bytes = smem_bytes<F8, NT>;
    static_assert(blocks_per_sm<NT> * (bytes + 1024) <= 228 * 1024, "shared memory of an SM");
    const cudaError_t e = q3_allow_shared_memory(tree_mma_kernel<F8, NT>, bytes, configured);
    if (e != cudaSuccess) return (int)e;
    using Work = TreeWork<PAGE, 8 * NT, false>;
    const int64_t units = Work::most_units(a.step, 0), most = (units + LEAST_PAGES - 1) / LEAST_PAGES + Work::most_items(a.step);
    if (Work::most_units(a.step, PART_PAGES) > 0x3fffffff) return Q3_ERR_TOO_LARGE;
    const int resident = blocks_per_sm<NT> * sm_count, grid = (int)(most < resident ? most : resident);
    return (int)q3_launch(tree_mma_kernel<F8, NT>, dim3(grid), dim3(WARPS * 32), (size_t)bytes, stream, a);
}
template <bool F8> int launch_rows(const Args& a, int64_t rows, cudaStream_t stream) {
    const int sms = q3_device_sm_count();
    return rows <= 8 ? launch<F8, 1>(a, sms, stream) : rows <= 16 ? launch<F8, 2>(a, sms, stream) : launch<F8, 4>(a, sms, stream);
}

}  // namespace

Q3_EXPORT int q3_attention_tree_mma_head_dim() { return D; }

// Float32 values of `parts` for a launch of up to so many rows (new tokens of a sequence x query heads a kv head); `counters`: one int32 for every
// sequence, kv head and 8 rows.
Q3_EXPORT int64_t q3_attention_tree_mma_parts(int rows) {
    const int each = rows <= 8 ? blocks_per_sm<1> * 8 : rows <= 16 ? blocks_per_sm<2> * 16 : blocks_per_sm<4> * 32;
    return (int64_t)2 * q3_device_sm_count() * each * (D + 2);
}

Q3_EXPORT int q3_attention_tree_mma_bf16(const q3_attention_tree_args* x) {
    if (x->n_seqs <= 0 || x->max_new <= 0) return 0;
    const int refused = tree_refused(*x, D);
    if (refused != 0) return refused;
    const Args a = {tree_step(*x), (const bf16*)x->q, (bf16*)x->out, (const unsigned char*)x->k_pages, (const unsigned char*)x->v_pages,
                    (const uint8_t*)x->k_scales, (const uint8_t*)x->v_scales, (float*)x->parts, (int*)x->counters, (float)x->scale * 1.4426950408889634f};
    const int64_t rows = (int64_t)x->max_new * (x->nq / x->nkv);
    return x->k_scales != nullptr ? launch_rows<true>(a, rows, (cudaStream_t)x->stream) : launch_rows<false>(a, rows, (cudaStream_t)x->stream);
}
