// Rows as 8-bit integers with a scale each: quantised as they are, or normed (after a residual sum) on the way.
//
// With a = max |x_k| of a row: code_k = 127 x_k / a to the nearest whole number, ties to even, and scale = a / 127.  The codes are those of the
// exact ratio: x_k is multiplied by the two 32-bit numbers next to 127 / a, below and above it, and where these round to different codes the middle
// between the two is compared with the ratio exactly (127 x_k against (code + 1/2) a, in 64 bits).  So every form, packet or thread layout gives the
// same codes, and a value that is not next to a tie costs two fused multiply-adds.
//
// The norm: t = x + delta (rounded to its type, and stored), y = t / sqrt(mean t^2 + eps) * w.  The root is common to a row, so it cancels
// from the codes: they are those of u = t * w (32 bits), and the scale is max |u| / sqrt(mean t^2 + eps) / 127.  The sum and the maximum
// go through one reduction, and a code does not hang on the order of the sum.
//
// A row with a NaN or an infinity (or whose squares' sum is none that 32 bits hold) gets the scale NaN and codes of zero: what is multiplied by it
// becomes NaN.  A row of zeros gets the scale zero.  Scales below 2^-126 have fewer bits.  An eps below 2^-126 (32 bits; zero, say) does not cover what
// squares of small values lose: rows whose mean square is below that are finished by a kernel of their own.
//
// Bound by memory: a row is read once, in packets of 16 bytes, held in registers across the reduction, and written (8,000 rows, of the measured copy
// rate: quantise 12,288 bfloat16 47.1 us, 0.95; 10,240 of 5,120 float32 42.5, 0.94; norm and sum 5,120 bfloat16 51, 0.86; in long runs, at the clocks that
// they settle at, 50.0, 48.2 and 56.1).  What a value
// costs in instructions comes next (seven in ten issue slots were taken where these times were 55 and 57): three-way maxima of packed halves, no
// fallbacks compiled into rows that need none, one rounding less and the scale's divisions in one thread took 10 and 6 %.  Blocks of up to 512 threads are bound to 64
// registers a thread, so that two fit an SM whatever their size; the variants that hold most (four packets of a norm, eight of float32 rows) spill 32 to 168 bytes a
// thread there, among them those that run the norm and the float32 rows above, in blocks of 160 threads; what they would take with more registers was not measured.
// Rows that do not begin at a packet's boundary (an odd width, a
// slice) are read in the packets around them, each thread shifting two into its own values: 5,001 bfloat16 24.4 and 76 us where 5,120 takes 20.8
// and 51.  Rows wider than 1,024 threads hold (32,768) are read twice, value by value: 400 of 70,001 bfloat16 45 us quantised and 135 normed, 3.5 and 4.5 times
// what their bytes take (no model here has them).  Tried and slower: rows brought several ahead by bulk copies into a ring in shared memory of blocks that stay (norm 5,120
// 126 us: barriers and a second pass over shared memory a row), 40 registers a thread for a third block (61.7), loads that are evicted first (1 to 2 %).
#include "common.cuh"
#include "../include/qwen3/int8_args.h"

namespace {

struct Rows {
    const void *x, *delta;
    const float* weight;
    void* total;
    int8_t* codes;
    float* scales;
    int64_t rows, x_stride, delta_stride, total_stride, codes_stride;
    int width;
    float eps, lost;                   // lost: a norm's sums of squares below this are taken again (0: none)
};

// What a row's codes are made with.
struct Grid {
    float top, ratio, below, above;    // max |u| (0: codes of zero), 127 / max |u| and the 32-bit numbers next to it
    bool divide;                       // a maximum so small that the ratio may not be finite: all codes divided out
};

__device__ __forceinline__ int code_exact(float u, const Grid& g) {
    if (g.divide) return __double2int_rn(__ddiv_rn(127.0 * (double)u, (double)g.top));     // (a quotient that is no tie is further from one than its rounding)
    const float low = floorf(u * g.below);
    const double over = 127.0 * (double)u - ((double)low + 0.5) * (double)g.top;           // exact: 31 and 32 bits
    const int k = (int)low;
    return over > 0.0 ? k + 1 : over < 0.0 ? k : k + (k & 1);
}

// Codes of N values, a byte each; four to a word.
template <int N> __device__ __forceinline__ void codes_of(const float (&u)[N], const Grid& g, uint32_t (&out)[N / 4]) {
    constexpr float MAGIC = 12582912.0f;                       // 1.5 * 2^23: adding it rounds to a whole number in the low bits
    uint32_t f[N], apart = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        f[i] = __float_as_uint(__fmaf_rn(u[i], g.below, MAGIC));
        apart |= f[i] ^ __float_as_uint(__fmaf_rn(u[i], g.above, MAGIC));
    }
    if (apart != 0u || g.divide) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (g.divide || f[i] != __float_as_uint(__fmaf_rn(u[i], g.above, MAGIC))) f[i] = (uint32_t)code_exact(u[i], g);
    }
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
        const uint32_t all = __byte_perm(__byte_perm(f[4 * w], f[4 * w + 1], 0x0040), __byte_perm(f[4 * w + 2], f[4 * w + 3], 0x0040), 0x5410);
        out[w] = g.top == 0.0f ? 0u : all;
    }
}

// The same for values of eight bits (bfloat16).  A ratio 127 x / a of two such numbers that is no tie is at least 1 / (256 * 253) from one at 1/2 and further
// from the others (every pair is in the tests), so rounding it to a multiple of 2^-15, as adding 384 does on either side of zero, moves no ratio onto a
// tie or over it, and brings a tie that the rounding of 127 / a has moved (by up to 2^-24 of itself) back onto it.
template <int N> __device__ __forceinline__ void codes_of_bf16(const float (&u)[N], const Grid& g, uint32_t (&out)[N / 4]) {
    if (g.divide) return codes_of<N>(u, g, out);
    uint32_t f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __float_as_uint(__fmaf_rn(u[i], g.ratio, 384.0f) + (12582912.0f - 384.0f));
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
        const uint32_t all = __byte_perm(__byte_perm(f[4 * w], f[4 * w + 1], 0x0040), __byte_perm(f[4 * w + 2], f[4 * w + 3], 0x0040), 0x5410);
        out[w] = g.top == 0.0f ? 0u : all;
    }
}

// `n` codes (of N) to a place that is a multiple of N bytes from the row's beginning.
template <int N, bool WHOLE> __device__ __forceinline__ void store_codes(int8_t* to, const uint32_t (&w)[N / 4], int n) {
    if constexpr (!WHOLE) {
        if (n < N) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < n) to[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
            return;
        }
    }
    if constexpr (N == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(to) = w[0];
}

template <typename T> __device__ __forceinline__ void unpack(const uint4& raw, float (&v)[Pack<T>::N]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            v[i] = __uint_as_float(w[i]);
        }
    }
}

// Where value c of a row lies; of 32-bit rows by a 32-bit offset from the row (in a row, with / without: 10,240 rows of 5,120 float32 quantised 47.4 / 49.5
// us, normed 101 / 103.5; bfloat16 rows normed 56.7 / 54).
template <typename T> __device__ __forceinline__ T* value_at(T* row, int c) {
    if constexpr (sizeof(T) == 4) return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(row) + (uint32_t)(c * 4));
    else return row + c;
}

// The packets of a row's values c .., zeros behind its end.  APART: rows may begin anywhere, and a packet of values lies in two packets of memory.  The
// first is asked for early (`fetch`) and held; the second is the next thread's first and is read when the two are shifted together (`whole`), from
// the L1 then.  Both have to lie inside the row, else the values are fetched one by one.
template <typename T, bool APART> struct Packet {
    static constexpr int N = Pack<T>::N;
    uint4 a;
    __device__ __forceinline__ void fetch(const T* row, int c, int width) {
        if constexpr (!APART) {
            a = c < width ? *reinterpret_cast<const uint4*>(value_at(row, c)) : make_uint4(0u, 0u, 0u, 0u);
        } else if (inside(c, width)) {
            a = *reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + c) & ~(uintptr_t)15);
        }
    }
    static __device__ __forceinline__ bool inside(int c, int width) { return c >= N && c + 2 * N <= width; }
    __device__ __forceinline__ uint4 whole(const T* row, int c, int width) const {
        if constexpr (!APART) return a;
        uint4 b = make_uint4(0u, 0u, 0u, 0u);
        if (inside(c, width)) b = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(row + c) & ~(uintptr_t)15)[1];
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;       // the same for all of the row's packets
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = off & 8u ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = off & 4u ? w[i + 1] : w[i];
        if constexpr (sizeof(T) == 2) {
            const uint32_t bits = (off & 2u) * 8u;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], bits);
        }
        if (!inside(c, width)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = 0u;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (c + i >= width) continue;
                if constexpr (sizeof(T) == 2) w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[c + i] << (16 * (i & 1));
                else w[i] = reinterpret_cast<const uint32_t*>(row)[c + i];
            }
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
// The norm's weights of values c .. (`whole`: all are there, at a 16-byte boundary).
template <int N> __device__ __forceinline__ void load_weights(const float* w, int c, int width, bool whole, float (&v)[N]) {
    if (whole) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 a = *reinterpret_cast<const float4*>(N == 4 ? value_at(w, c) : w + c + i);        // (N 4: rows of 32 bits)
            v[i] = a.x; v[i + 1] = a.y; v[i + 2] = a.z; v[i + 3] = a.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = c + i < width ? w[c + i] : 0.0f;
    }
}

// The largest magnitude as bits: an infinity's or NaN's are above every finite number's.
template <typename T> __device__ __forceinline__ uint32_t top_of(const uint4& raw, uint32_t top) {
    constexpr uint32_t M = sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu;
    if constexpr (sizeof(T) == 2) return __vimax3_u16x2(__vimax3_u16x2(top, raw.x & M, raw.y & M), raw.z & M, raw.w & M);
    else return __vimax3_u32(__vimax3_u32(top, raw.x & M, raw.y & M), raw.z & M, raw.w & M);
}
// (of two 16-bit halves the larger one, as 32 bits)
template <typename T> __device__ __forceinline__ uint32_t top_bits(uint32_t top) {
    return sizeof(T) == 2 ? max(top << 16, top & 0xffff0000u) : top;
}

// The largest magnitude and the sum of squares over a row's threads.
template <bool WARP, bool NORM> __device__ __forceinline__ void reduce(uint32_t& top, float& squares) {
    top = __reduce_max_sync(0xffffffffu, top);
    if (NORM) squares = warp_sum(squares);
    if constexpr (!WARP) {
        __shared__ uint32_t tops[32];
        __shared__ float sums[32];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0) {
            tops[warp] = top;
            sums[warp] = squares;
        }
        __syncthreads();
        const bool in = lane < (int)(blockDim.x >> 5);
        top = __reduce_max_sync(0xffffffffu, in ? tops[lane] : 0u);
        if (NORM) squares = warp_sum(in ? sums[lane] : 0.0f);
    }
}

// What the codes are made with; the row's first thread writes the scale, whose root and divisions the others do without.
template <bool NORM> __device__ __forceinline__ Grid finish(const Rows& a, int64_t row, bool first, uint32_t bits, float squares) {
    const float top = __uint_as_float(bits);
    bool fine = bits < 0x7f800000u;
    if constexpr (NORM) fine = fine && squares < INFINITY;
    if (first)
        a.scales[row] = !fine ? __uint_as_float(0x7fffffffu)
                        : !NORM || top == 0.0f ? top / 127.0f
                        : squares < a.lost ? -top              // (for `small_rows_kernel`)
                                           : top * rsqrtf(squares / (float)a.width + a.eps) / 127.0f;
    Grid g;
    g.top = fine ? top : 0.0f;
    g.divide = g.top != 0.0f && top < 7.9e-31f;                // 2^-100
    g.ratio = __fdiv_rn(127.0f, fmaxf(top, 7.9e-31f));
    g.below = __uint_as_float(__float_as_uint(g.ratio) - 1u);
    g.above = __uint_as_float(__float_as_uint(g.ratio) + 1u);
    return g;
}

// A packet of sums to where they are stored: at once, or, where rows may begin anywhere, through shared memory: a warp's 32 packets are consecutive
// values, which go out side by side.
template <typename T, bool APART> __device__ __forceinline__ void store_total(T* row, int c, int width, const uint4& k) {
    constexpr int N = Pack<T>::N;
    if constexpr (!APART) {
        if (c < width) *reinterpret_cast<uint4*>(value_at(row, c)) = k;
    } else {
        extern __shared__ __align__(16) unsigned char staged[];
        const int lane = threadIdx.x & 31, first = c - lane * N;
        T* mine = reinterpret_cast<T*>(staged) + (threadIdx.x >> 5) * (32 * N);
        __syncwarp();
        *reinterpret_cast<uint4*>(mine + lane * N) = k;
        __syncwarp();
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (first + i * 32 + lane < width) row[first + i * 32 + lane] = mine[i * 32 + lane];
        } else {                                               // words of two values where they lie on word boundaries
            const int odd = (int)(reinterpret_cast<uintptr_t>(row) >> 1) & 1, live = min(32 * N, width - first);
            const uint16_t* from = reinterpret_cast<const uint16_t*>(mine);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const int at = 2 * (i * 32 + lane) + odd;
                if (at + 1 < live) *reinterpret_cast<uint32_t*>(row + first + at) = (uint32_t)from[at] | (uint32_t)from[at + 1] << 16;
                else if (at < live) row[first + at] = mine[at];
            }
            if (odd && lane == 0 && live > 0) row[first] = mine[0];
        }
    }
}

// x + delta of a packet, rounded to the type.
template <typename T> __device__ __forceinline__ uint4 sum_of(const uint4& x, const uint4& d) {
    const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {d.x, d.y, d.z, d.w};
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(__uint_as_float(a[i] << 16) + __uint_as_float(b[i] << 16),
                                                           __uint_as_float(a[i] & 0xffff0000u) + __uint_as_float(b[i] & 0xffff0000u));
            w[i] = *reinterpret_cast<const uint32_t*>(&t);
        } else {
            w[i] = __float_as_uint(__uint_as_float(a[i]) + __uint_as_float(b[i]));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row a block, or (WARP) a row a warp; a thread holds PER packets.  Of a norm it holds the products with the weights, or (rows of bfloat16 at packet
// boundaries) the sums as they are stored, in half the registers, and makes the products twice (the other way round / so: 8,000 rows of 5,120
// bfloat16 51.9 / 50.8 us, of 5,001 77.0 / 84.8, of 4,097 float32 103.8 / 111.6).
template <typename T, int PER, bool NORM, bool APART, bool WARP, int MOST_THREADS>
__global__ void __launch_bounds__(MOST_THREADS, MOST_THREADS == 512 ? 2 : 1) rows_kernel(const Rows a) {
    constexpr int N = Pack<T>::N;
    pdl_wait();
    pdl_launch_dependents();
    const int threads = WARP ? 32 : blockDim.x, thread = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= a.rows) return;
    const T* x = (const T*)a.x + row * a.x_stride;
    const bool whole_weights = NORM && (reinterpret_cast<uintptr_t>(a.weight) & 15u) == 0;
    Packet<T, APART> from_x[PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) from_x[p].fetch(x, (p * threads + thread) * N, a.width);
    constexpr bool HOLD = NORM && (APART || sizeof(T) == 4);
    uint4 raw[PER];
    float held[HOLD ? PER : 1][N];
    if (NORM && a.delta != nullptr) {
        const T* delta = (const T*)a.delta + row * a.delta_stride;
        T* total = (T*)a.total + row * a.total_stride;
        Packet<T, APART> from_delta[PER];
#pragma unroll
        for (int p = 0; p < PER; ++p) from_delta[p].fetch(delta, (p * threads + thread) * N, a.width);
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int c = (p * threads + thread) * N;
            raw[p] = sum_of<T>(from_x[p].whole(x, c, a.width), from_delta[p].whole(delta, c, a.width));
            store_total<T, APART>(total, c, a.width, raw[p]);
        }
    } else {
#pragma unroll
        for (int p = 0; p < PER; ++p) raw[p] = from_x[p].whole(x, (p * threads + thread) * N, a.width);
    }
    float squares = 0.0f;
    uint32_t top = 0u;
    auto weighted = [&](int p, int c, float (&u)[N]) {         // what the codes are made of
        unpack<T>(raw[p], u);
        if constexpr (NORM) {
            float w[N];
            load_weights<N>(a.weight, c, a.width, !APART || (whole_weights && c + N <= a.width), w);
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] *= w[i];
        }
    };
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int c = (p * threads + thread) * N;
        if constexpr (!NORM) {
            top = top_of<T>(raw[p], top);
        } else if (c < a.width) {
            float t[N], u[N];
            unpack<T>(raw[p], t);
            weighted(p, c, u);
            if constexpr (HOLD) {
#pragma unroll
                for (int i = 0; i < N; ++i) held[p][i] = u[i];
            }
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                squares += t[i] * t[i];
                squares += t[i + 1] * t[i + 1];
                top = __vimax3_u32(top, __float_as_uint(u[i]) & 0x7fffffffu, __float_as_uint(u[i + 1]) & 0x7fffffffu);
            }
        }
    }
    if (!NORM) top = top_bits<T>(top);
    reduce<WARP, NORM>(top, squares);
    const Grid g = finish<NORM>(a, row, thread == 0, top, squares);
    int8_t* codes = a.codes + row * a.codes_stride;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int c = (p * threads + thread) * N;
        if (c >= a.width) continue;
        uint32_t w[N / 4];
        float u[N];
        if constexpr (HOLD) {
#pragma unroll
            for (int i = 0; i < N; ++i) u[i] = held[p][i];
        } else {
            weighted(p, c, u);
        }
        if constexpr (sizeof(T) == 2 && !NORM) codes_of_bf16<N>(u, g, w);
        else codes_of<N>(u, g, w);
        store_codes<N, !APART>(codes + (uint32_t)c, w, a.width - c);
    }
}

// A row that does not fit the registers of a block: read twice, four values at a time.
template <typename T, bool NORM> __global__ void __launch_bounds__(1024) long_rows_kernel(const Rows a) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    float squares = 0.0f, u[4];
    uint32_t top = 0u;
    auto values = [&](int c, bool store) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u[i] = c + i < a.width ? to_f32<T>(x[c + i]) : 0.0f;
            if constexpr (NORM) {
                if (c + i >= a.width) continue;
                if (a.delta != nullptr) {
                    u[i] = round_to<T>(u[i] + to_f32<T>(((const T*)a.delta)[row * a.delta_stride + c + i]));
                    if (store) ((T*)a.total)[row * a.total_stride + c + i] = from_f32<T>(u[i]);
                }
                squares += u[i] * u[i];
                u[i] *= a.weight[c + i];
            }
        }
    };
    for (int c = threadIdx.x * 4; c < a.width; c += 4096) {
        values(c, false);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(u[i]) & 0x7fffffffu);
    }
    reduce<false, NORM>(top, squares);
    const Grid g = finish<NORM>(a, row, threadIdx.x == 0, top, squares);
    for (int c = threadIdx.x * 4; c < a.width; c += 4096) {
        values(c, true);                                       // (the sum is stored now: `total` may be x)
        uint32_t w[1];
        codes_of<4>(u, g, w);
        store_codes<4, false>(a.codes + row * a.codes_stride + c, w, a.width - c);
    }
}

// The scales of normed rows whose squares 32 bits lose, after one of the kernels above has noted -max |u| in their place: a row a warp, sums in 64 bits, which
// hold the square of every 32-bit number.
template <typename T> __global__ void __launch_bounds__(256) small_rows_kernel(const Rows a) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= a.rows) return;
    const float noted = a.scales[row];
    if (!(noted < 0.0f)) return;
    const T* t = a.delta != nullptr ? (const T*)a.total + row * a.total_stride : (const T*)a.x + row * a.x_stride;
    double squares = 0.0;
    for (int64_t c = lane; c < a.width; c += 32) {
        const double v = (double)to_f32<T>(t[c]);
        squares += v * v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    if (lane == 0) a.scales[row] = (float)(-(double)noted / sqrt(squares / (double)a.width + (double)a.eps) / 127.0);
}

template <typename T, int PER, bool NORM, bool APART> int launch(const Rows& a, int threads, bool warp, cudaStream_t stream) {
    const int block = warp ? 128 : threads;
    const size_t staged = NORM && APART && a.delta != nullptr ? (size_t)block * 16 : 0;
    if (warp)
        return (int)q3_launch(rows_kernel<T, PER, NORM, APART, true, 128>, dim3((unsigned)((a.rows + 3) / 4)), dim3(block), staged, stream, a);
    if (threads <= 512) return (int)q3_launch(rows_kernel<T, PER, NORM, APART, false, 512>, dim3((unsigned)a.rows), dim3(block), staged, stream, a);
    return (int)q3_launch(rows_kernel<T, PER, NORM, APART, false, 1024>, dim3((unsigned)a.rows), dim3(block), staged, stream, a);
}

template <typename T, bool NORM, bool APART> int pick(const Rows& a, cudaStream_t stream) {
    constexpr int N = Pack<T>::N, MOST = 32 / N;               // packets that a thread may hold
    const int packets = (a.width + N - 1) / N;
    const int64_t sms = q3_device_sm_count();
    // short rows, if they are many: a row a warp
    const bool warp = a.rows >= 2 * sms && packets <= 32 * MOST;
    // As few packets a thread as the SMs can hold threads for at once: few rows want threads, many want loads in flight while other rows of the SM are
    // reduced.  (8,000 rows of 4,096, bfloat16, 4 / 2 / 1 packets a thread, when it was measured: norm 42.8 / 47.9 / 66 us, quantise 17.7 / 21.7 / 29.3; 527 rows
    // 6.6 / 4.7 / 5.5 and 3.2 / 2.6 / 2.7.  float32 8 / 4: quantise 8,000 rows of 5,120 36.2 / 41.4, of 4,097 49.5 / 43.0, norm 100 / 81.)
    int per = 1;
    if (warp) {
        while (32 * per < packets) per *= 2;
    } else {
        while (per < (NORM || APART ? 4 : MOST) && a.rows * ((packets + per - 1) / per) > 1200 * sms) per *= 2;
        while (per < MOST && packets > 1024 * per) per *= 2;
    }
    const int threads = ((packets + per - 1) / per + 31) / 32 * 32;
    if (threads > 1024) return (int)q3_launch(long_rows_kernel<T, NORM>, dim3((unsigned)a.rows), dim3(1024), 0, stream, a);
    if (per == 1) return launch<T, 1, NORM, APART>(a, threads, warp, stream);
    if (per == 2) return launch<T, 2, NORM, APART>(a, threads, warp, stream);
    if (per == 4) return launch<T, 4, NORM, APART>(a, threads, warp, stream);
    return launch<T, MOST, NORM, APART>(a, threads, warp, stream);
}

template <typename T, bool NORM> int rows_launch(const q3_int8_rows_args& in) {
    constexpr int V = Pack<T>::N;
    if (in.rows <= 0 || in.width < 0) return in.rows < 0 || in.width < 0 ? Q3_ERR_BAD_SIZE : 0;
    if (in.width == 0) return (int)cudaMemsetAsync(in.scales, 0, (size_t)in.rows * sizeof(float), (cudaStream_t)in.stream);     // as a row of zeros
    if (in.rows > 0x7fffffff || in.width > 1 << 30) return Q3_ERR_TOO_LARGE;
    if (in.codes_stride < in.width || in.x == nullptr || (NORM && (in.weight == nullptr || (in.delta != nullptr && in.total == nullptr))))
        return Q3_ERR_BAD_SIZE;
    if (in.codes_stride % 16 != 0 || !aligned16(in.codes)) return Q3_ERR_MISALIGNED;
    const Rows a{in.x, NORM ? in.delta : nullptr, NORM ? (const float*)in.weight : nullptr, NORM ? in.total : nullptr, (int8_t*)in.codes,
                 (float*)in.scales, in.rows, in.x_stride, in.delta_stride, in.total_stride, in.codes_stride, in.width, (float)in.eps,
                 NORM && (float)in.eps < 0x1p-126f ? (float)in.width * 0x1p-126f : 0.0f};
    const bool packets = in.width % V == 0 && in.x_stride % V == 0 && aligned16(in.x) && aligned16(a.weight) &&
                         (a.delta == nullptr || (in.delta_stride % V == 0 && in.total_stride % V == 0 && aligned16(in.delta) && aligned16(in.total)));
    const cudaStream_t stream = (cudaStream_t)in.stream;
    const int failed = packets ? pick<T, NORM, false>(a, stream) : pick<T, NORM, true>(a, stream);
    if constexpr (NORM)
        if (failed == 0 && a.lost > 0.0f) return (int)q3_launch(small_rows_kernel<T>, dim3((unsigned)((a.rows + 7) / 8)), dim3(256), 0, stream, a);
    return failed;
}

}  // namespace

Q3_EXPORT int q3_quantize_rows_f32(const q3_int8_rows_args* a) { return rows_launch<float, false>(*a); }
Q3_EXPORT int q3_quantize_rows_bf16(const q3_int8_rows_args* a) { return rows_launch<bf16, false>(*a); }
Q3_EXPORT int q3_rms_norm_int8_f32(const q3_int8_rows_args* a) { return rows_launch<float, true>(*a); }
Q3_EXPORT int q3_rms_norm_int8_bf16(const q3_int8_rows_args* a) { return rows_launch<bf16, true>(*a); }
