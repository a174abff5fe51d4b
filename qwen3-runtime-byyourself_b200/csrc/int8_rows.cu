// Rows as 8-bit integers with a scale each: quantised as they are, or normed (after a residual sum) on the way.
//
// With a = max |x_k| of a row: code_k = 127 x_k / a to the nearest whole number, ties to even, and scale = a / 127.  The codes are those of the
// exact ratio: a product with 127 / a decides unless it comes within 2^-15 of the middle between two codes, where the ratio is divided out in
// 64 bits (127 x is exact there, and a quotient that is no tie is further from one than its rounding).  So every form, packet or thread layout gives the
// same codes.
//
// The norm: t = x + delta (rounded to its type, and stored), y = t / sqrt(mean t^2 + eps) * w.  The root is common to a row, so it cancels
// from the codes: they are those of u = t * w (32 bits), and the scale is max |u| / sqrt(mean t^2 + eps) / 127.  The sum and the maximum
// go through one reduction, and a code does not hang on the order of the sum.
//
// A row with a NaN or an infinity (or whose squares' sum is none that 32 bits hold) gets the scale NaN and codes of zero: what is multiplied by it
// becomes NaN.  A row of zeros gets the scale zero.  Scales below 2^-126 have fewer bits.
//
// Bound by memory: a row is read once, held in registers across the reduction, and written.
#include "common.cuh"
#include "../include/qwen3/int8_args.h"

namespace {

constexpr int MOST = 32;               // values of a row that a thread holds

struct Rows {
    const void *x, *delta;
    const float* weight;
    void* total;
    int8_t* codes;
    float* scales;
    int64_t rows, x_stride, delta_stride, total_stride, codes_stride;
    int width;
    float eps;
};

// What a row's codes are made with.
struct Grid {
    float top, ratio;                  // max |u| (0: codes of zero) and 127 / max |u|
    bool exact;                        // a maximum so small that the ratio may not be finite: all codes divided out
};

__device__ __forceinline__ int code_exact(float u, float top) { return __double2int_rn(__ddiv_rn(127.0 * (double)u, (double)top)); }

// Codes of N values, a byte each; four to a word.
template <int N> __device__ __forceinline__ void codes_of(const float (&u)[N], const Grid& g, uint32_t (&out)[(N + 3) / 4]) {
    constexpr float MAGIC = 12582912.0f;                       // 1.5 * 2^23: adding it rounds to a whole number in the low bits
    float f[N], worst = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float q = u[i] * g.ratio;
        f[i] = q + MAGIC;
        worst = fmaxf(worst, fabsf(q - (f[i] - MAGIC)));
    }
    if (worst > 0.5f - 1.0f / 32768.0f || g.exact) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float q = u[i] * g.ratio;
            if (g.exact || fabsf(q - (f[i] - MAGIC)) > 0.5f - 1.0f / 32768.0f) f[i] = MAGIC + (float)code_exact(u[i], g.top);
        }
    }
#pragma unroll
    for (int w = 0; w < (N + 3) / 4; ++w) {
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = 4 * w + i < N ? __float_as_uint(f[4 * w + i < N ? 4 * w + i : 0]) : 0u;
        out[w] = g.top == 0.0f ? 0u : __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
}

template <int VEC> __device__ __forceinline__ void store_codes(int8_t* to, const uint32_t (&w)[(VEC + 3) / 4]) {
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(to) = w[0];
    else to[0] = (int8_t)(w[0] & 0xffu);
}

template <typename T, int VEC> __device__ __forceinline__ void load_values(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = to_f32<T>(p[0]);
    } else {
        const Pack<T> k = load_pack<T>(p);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = k.get(i);
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_values(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        p[0] = from_f32<T>(v[0]);
    } else {
        Pack<T> k;
#pragma unroll
        for (int i = 0; i < VEC; ++i) k.set(i, v[i]);
        store_pack<T>(p, k);
    }
}
template <int VEC> __device__ __forceinline__ void load_weights(const float* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = p[0];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 w = *reinterpret_cast<const float4*>(p + i);
            v[i] = w.x; v[i + 1] = w.y; v[i + 2] = w.z; v[i + 3] = w.w;
        }
    }
}

// Values c .. c + VEC - 1 of a row as they go into the codes; adds to the sum of squares.
template <typename T, int VEC, bool NORM>
__device__ __forceinline__ void values_of(const Rows& a, int64_t row, int c, float (&u)[VEC], float& squares, bool store) {
    load_values<T, VEC>((const T*)a.x + row * a.x_stride + c, u);
    if constexpr (NORM) {
        if (a.delta != nullptr) {
            float d[VEC];
            load_values<T, VEC>((const T*)a.delta + row * a.delta_stride + c, d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) u[i] = round_to<T>(u[i] + d[i]);
            if (store) store_values<T, VEC>((T*)a.total + row * a.total_stride + c, u);
        }
        float w[VEC];
        load_weights<VEC>(a.weight + c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            squares += u[i] * u[i];
            u[i] *= w[i];
        }
    }
}

// The largest magnitude (as bits: above every finite number's where there is an infinity or NaN) and the sum of squares over a row's threads.
template <bool WARP> __device__ __forceinline__ void reduce(uint32_t& top, float& squares, bool norm) {
    top = __reduce_max_sync(0xffffffffu, top);
    if (norm) squares = warp_sum(squares);
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
        if (norm) squares = warp_sum(in ? sums[lane] : 0.0f);
    }
}

template <bool NORM> __device__ __forceinline__ Grid finish(const Rows& a, uint32_t top_bits, float squares, float& scale) {
    const float top = __uint_as_float(top_bits);
    float mean = 0.0f;
    bool fine = top_bits < 0x7f800000u;
    if constexpr (NORM) {
        mean = squares / (float)a.width;
        fine = fine && mean < INFINITY;
    }
    scale = !fine ? __uint_as_float(0x7fffffffu) : NORM ? top * rsqrtf(mean + a.eps) / 127.0f : top / 127.0f;
    Grid g;
    g.top = fine ? top : 0.0f;
    g.exact = top < 7.9e-31f;                                  // 2^-100
    g.ratio = __fdiv_rn(127.0f, fmaxf(top, 7.9e-31f));
    return g;
}

// A row a block, or (WARP) a row a warp; a thread holds PER packets of VEC values.
template <typename T, int VEC, int PER, bool NORM, bool WARP>
__global__ void __launch_bounds__(WARP ? 128 : 1024) rows_kernel(const Rows a) {
    pdl_launch_dependents();
    pdl_wait();
    const int threads = WARP ? 32 : blockDim.x, thread = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = WARP ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= a.rows) return;
    float u[PER][VEC], squares = 0.0f;
    uint32_t top = 0u;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int c = (p * threads + thread) * VEC;
        if (c < a.width) {
            values_of<T, VEC, NORM>(a, row, c, u[p], squares, true);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) u[p][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) top = max(top, __float_as_uint(u[p][i]) & 0x7fffffffu);
    }
    reduce<WARP>(top, squares, NORM);
    float scale;
    const Grid g = finish<NORM>(a, top, squares, scale);
    if (thread == 0) a.scales[row] = scale;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
        const int c = (p * threads + thread) * VEC;
        if (c < a.width) {
            uint32_t w[(VEC + 3) / 4];
            codes_of<VEC>(u[p], g, w);
            store_codes<VEC>(a.codes + row * a.codes_stride + c, w);
        }
    }
}

// A row that does not fit the registers of a block: read twice.
template <typename T, bool NORM> __global__ void __launch_bounds__(1024) long_rows_kernel(const Rows a) {
    pdl_launch_dependents();
    pdl_wait();
    const int64_t row = blockIdx.x;
    float squares = 0.0f, u[1];
    uint32_t top = 0u;
    for (int c = threadIdx.x; c < a.width; c += 1024) {
        values_of<T, 1, NORM>(a, row, c, u, squares, false);
        top = max(top, __float_as_uint(u[0]) & 0x7fffffffu);
    }
    reduce<false>(top, squares, NORM);
    float scale, unused = 0.0f;
    const Grid g = finish<NORM>(a, top, squares, scale);
    if (threadIdx.x == 0) a.scales[row] = scale;
    for (int c = threadIdx.x; c < a.width; c += 1024) {
        values_of<T, 1, NORM>(a, row, c, u, unused, true);     // (the sum is stored now: `total` may be x)
        uint32_t w[1];
        codes_of<1>(u, g, w);
        store_codes<1>(a.codes + row * a.codes_stride + c, w);
    }
}

template <typename T, int VEC, int PER, bool NORM> int launch(const Rows& a, int threads, bool warp, cudaStream_t stream) {
    if (warp)
        return (int)q3_launch(rows_kernel<T, VEC, PER, NORM, true>, dim3((unsigned)((a.rows + 3) / 4)), dim3(128), 0, stream, a);
    return (int)q3_launch(rows_kernel<T, VEC, PER, NORM, false>, dim3((unsigned)a.rows), dim3(threads), 0, stream, a);
}

template <typename T, int VEC, bool NORM> int pick(const Rows& a, cudaStream_t stream) {
    const int packets = (a.width + VEC - 1) / VEC, most = MOST / VEC;
    const bool many = a.rows >= 2 * q3_device_sm_count();
    const bool warp = many && packets <= 32 * most;
    int per = warp ? (packets + 31) / 32 : many ? (packets + 255) / 256 : (packets + 1023) / 1024;
    if (per > most) per = most;
    int p = VEC == 1 ? 4 : 1;                                  // packets a thread: the next power of two
    while (p < per) p *= 2;
    const int threads = ((packets + p - 1) / p + 31) / 32 * 32;
    if (threads > 1024)
        return (int)q3_launch(long_rows_kernel<T, NORM>, dim3((unsigned)a.rows), dim3(1024), 0, stream, a);
    switch (p * VEC) {
        case 4: return launch<T, VEC, (4 / VEC > 0 ? 4 / VEC : 1), NORM>(a, threads, warp, stream);
        case 8: return launch<T, VEC, 8 / VEC, NORM>(a, threads, warp, stream);
        case 16: return launch<T, VEC, 16 / VEC, NORM>(a, threads, warp, stream);
        default: return launch<T, VEC, 32 / VEC, NORM>(a, threads, warp, stream);
    }
}

template <typename T, bool NORM> int rows_launch(const q3_int8_rows_args& in) {
    constexpr int V = Pack<T>::N;
    if (in.rows <= 0 || in.width <= 0) return in.rows < 0 || in.width < 0 ? Q3_ERR_BAD_SIZE : 0;
    if (in.rows > 0x7fffffff) return Q3_ERR_TOO_LARGE;
    if (in.codes_stride < in.width || in.x == nullptr || (NORM && (in.weight == nullptr || (in.delta != nullptr && in.total == nullptr))))
        return Q3_ERR_BAD_SIZE;
    if (in.codes_stride % 16 != 0 || !aligned16(in.codes)) return Q3_ERR_MISALIGNED;
    const Rows a{in.x, NORM ? in.delta : nullptr, NORM ? (const float*)in.weight : nullptr, NORM ? in.total : nullptr, (int8_t*)in.codes,
                 (float*)in.scales, in.rows, in.x_stride, in.delta_stride, in.total_stride, in.codes_stride, in.width, (float)in.eps};
    const bool packets = in.width % V == 0 && in.x_stride % V == 0 && aligned16(in.x) &&
                         (!NORM || (aligned16(in.weight) && (in.delta == nullptr || (in.delta_stride % V == 0 && in.total_stride % V == 0 &&
                                                                                      aligned16(in.delta) && aligned16(in.total)))));
    return packets ? pick<T, V, NORM>(a, (cudaStream_t)in.stream) : pick<T, 1, NORM>(a, (cudaStream_t)in.stream);
}

}  // namespace

Q3_EXPORT int q3_quantize_rows_f32(const q3_int8_rows_args* a) { return rows_launch<float, false>(*a); }
Q3_EXPORT int q3_quantize_rows_bf16(const q3_int8_rows_args* a) { return rows_launch<bf16, false>(*a); }
Q3_EXPORT int q3_rms_norm_int8_f32(const q3_int8_rows_args* a) { return rows_launch<float, true>(*a); }
Q3_EXPORT int q3_rms_norm_int8_bf16(const q3_int8_rows_args* a) { return rows_launch<bf16, true>(*a); }
