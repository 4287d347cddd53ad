// Rows of activations to int8 with one scale a row: behind the residual's addition and the RMSNorm, or as they are.
//
// With u[c] = x[c] (1 + w[c]) col_scale[c] and r = 1 / sqrt(mean(x^2) + eps) the normed row is v = r u, r > 0. Then max |v| = r max |u| and
// v / max |v| = u / max |u|: the bytes do not depend on r at all, only the row's scale does. So the sum of squares and the maximum are taken
// in ONE pass over the registers and the block meets at one barrier, where norm, then maximum, then rounding would meet at two.
//
// What bounds it: memory (3 to 13 bytes a value, under ten instructions). A block owns a row and keeps it in registers between the
// reduction and the rounding, a thread up to four vectors of 16 bytes (a 2560-wide float32 row is 160 threads, a 9728-wide binary16 row
// 320), all of whose loads are issued before the first is used and leave the L1 to the gains. With two vectors to a thread a single row
// is 0.3 us faster and 4096 rows of 4096 values 3.6 us slower (23.1 and 19.5); a ring of rows in shared memory, filled by bulk copies
// while groups of warps round, was built and was 10 to 30 % slower but for 48 KB rows without gains, and persistent blocks that load their
// next row while they reduce one were level at best. Rows wider than 768 threads hold are
// read again behind the barrier (from the L2). Rows that are not aligned to the vectors, or whose length is odd, take a kernel of single-value
// accesses. Measured alone, back to back, against the memory's 6.56 TB/s: 4096 x 2560, float32 delta 24.1 us (86 %), binary16 delta 20.5 (86 %);
// 4096 x 4096 without 19.5 (66 %); quantise 4096 x 9728 binary16 22.9 (80 %), 4096 x 12288 float32 46.1 (83 %); 900 x 2560, binary16 delta 7.0
// (55 %: half of it a launch's start and end); one row 2.1 to 2.6 us.
#include "rows_s8.hpp"

#include <cmath>
#include <cstdint>
#include <stdexcept>
#include <string>

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "context.hpp"
#include "ptx.cuh"

namespace sepal::b200 {

void count_launch();

namespace {

constexpr int kHeld = 4;                 // vectors a thread keeps
constexpr unsigned kMaxThreads = 768, kNarrowThreads = 512;
constexpr unsigned kInfBits = 0x7F800000u;

struct RowsParams {
    const void* x;  // the norm's float32 stream is also written
    std::size_t ld_x;
    const void* delta;
    std::size_t ld_delta;
    const float* w;
    const float* col_scale;
    std::int8_t* q;
    std::size_t ld_q;
    float* scales;
    __half* values;  // or null
    std::size_t ld_values;
    std::size_t cols;
    float eps;
};

// Both forms give a row to the same number of threads, thread i the vectors i, i + threads, ..., and adds the threads' sums in the same order:
// a row's scale has the same bits whichever form its call took.
//
// What the block's threads make of a row: the sum of x^2 and the largest |u| as the bit pattern of a non-negative float, which orders like
// an unsigned integer, infinities and NaN last. One barrier.
template <bool NORM>
__device__ __forceinline__ void reduce_row(float& sum, unsigned& top) {
    __shared__ float sums[kMaxThreads / 32];
    __shared__ unsigned tops[kMaxThreads / 32];
    const unsigned warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    top = __reduce_max_sync(0xFFFFFFFFu, top);
    if constexpr (NORM) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
    if (warps == 1) return;
    if (lane == 0) {
        tops[warp] = top;
        if constexpr (NORM) sums[warp] = sum;
    }
    __syncthreads();
    top = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? tops[lane] : 0u);
    if constexpr (NORM) {
        sum = lane < warps ? sums[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
}

// The row's scale, and the factors its values are multiplied by before they are rounded: u * lift * inv. (127 / top overflows for a top under
// 2^-121; lifted by 2^64, which is exact, it does not. lift is 1 otherwise, so that inv is the 127 / max of launch_quantize_rows_s8.)
struct RowScale {
    float scale, lift, inv;
    bool finite;
};
template <bool NORM>
__device__ __forceinline__ RowScale row_scale(float sum, unsigned top_bits, const RowsParams& p) {
    RowScale s;
    const float top = __uint_as_float(top_bits);
    s.lift = top < 0x1p-64f ? 0x1p64f : 1.0f;
    s.inv = top > 0.0f ? __fdiv_rn(127.0f, __fmul_rn(top, s.lift)) : 0.0f;
    float scaled = top;
    if constexpr (NORM) scaled = __fdiv_rn(top, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.cols)), p.eps)));
    // max |v| itself: it may overflow where max |u| did not. (NaN compares false; squares that overflow would leave a maximum of 0.)
    s.finite = scaled < __uint_as_float(kInfBits) && (!NORM || sum < __uint_as_float(kInfBits));
    s.scale = s.finite ? __fdiv_rn(scaled, 127.0f) : __uint_as_float(0x7FC00000u);
    return s;
}

// Round to nearest even by adding 1.5 * 2^23: |u lift inv| is at most 127 (1 + 2^-23), so the low byte of the sum is the integer in two's
// complement, and the sum less 1.5 * 2^23 the integer itself. One addition where a conversion runs at a quarter of the rate.
constexpr float kRound = 12582912.0f;
__device__ __forceinline__ float rounded(float u, const RowScale& s) { return __fadd_rn(__fmul_rn(__fmul_rn(u, s.lift), s.inv), kRound); }
__device__ __forceinline__ unsigned byte_of(float r) { return __float_as_uint(r) & 0xFFu; }
// What a byte stands for, in binary16: one float32 product, rounded once more.
__device__ __forceinline__ __half value_of(float r, const RowScale& s) { return __float2half_rn(__fmul_rn(__fsub_rn(r, kRound), s.scale)); }

// N consecutive results, four or eight: one store of their bytes, and one of their values where they are asked for.
template <bool VALUES, int N>
__device__ __forceinline__ void store_vector(const RowsParams& p, std::size_t row, unsigned vec, const float (&u)[N], const RowScale& s) {
    unsigned bytes[N / 4], halves[N / 2];
    if (!s.finite) {  // (the whole block's)
#pragma unroll
        for (int h = 0; h < N / 4; ++h) bytes[h] = 0u, halves[2 * h] = halves[2 * h + 1] = 0x7FFF7FFFu;
    } else {
#pragma unroll
        for (int h = 0; h < N / 4; ++h) {
            float r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = rounded(u[4 * h + j], s);
            bytes[h] = __byte_perm(__byte_perm(__float_as_uint(r[0]), __float_as_uint(r[1]), 0x0040), __byte_perm(__float_as_uint(r[2]), __float_as_uint(r[3]), 0x0040), 0x5410);
            if constexpr (VALUES) {
                const __half2 lo = __halves2half2(value_of(r[0], s), value_of(r[1], s)), hi = __halves2half2(value_of(r[2], s), value_of(r[3], s));
                halves[2 * h] = *reinterpret_cast<const unsigned*>(&lo), halves[2 * h + 1] = *reinterpret_cast<const unsigned*>(&hi);
            }
        }
    }
    std::int8_t* const q = p.q + row * p.ld_q;
    if constexpr (N == 8) {
        reinterpret_cast<uint2*>(q)[vec] = make_uint2(bytes[0], bytes[1]);
        if constexpr (VALUES) reinterpret_cast<uint4*>(p.values + row * p.ld_values)[vec] = make_uint4(halves[0], halves[1], halves[2], halves[3]);
    } else {
        reinterpret_cast<unsigned*>(q)[vec] = bytes[0];
        if constexpr (VALUES) reinterpret_cast<uint2*>(p.values + row * p.ld_values)[vec] = make_uint2(halves[0], halves[1]);
    }
}

__device__ __forceinline__ void widen(const uint4& raw, float (&v)[8]) {
    const unsigned bits[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&bits[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ float4 product(const float4& a, const float4& b) {
    return make_float4(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y), __fmul_rn(a.z, b.z), __fmul_rn(a.w, b.w));
}
__device__ __forceinline__ float square_into(float sum, const float4& v) {
    return __fmaf_rn(v.w, v.w, __fmaf_rn(v.z, v.z, __fmaf_rn(v.y, v.y, __fmaf_rn(v.x, v.x, sum))));
}
// 16 bytes that are read once: they leave the L1 to the gains, which every row reads again.
__device__ __forceinline__ uint4 load_once(const void* at) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 load_once_f32(const void* at) {
    const uint4 v = load_once(at);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

__device__ __forceinline__ unsigned largest_of(unsigned top, const float4& u) {
    return max(max(top, max(magnitude(u.x), magnitude(u.y))), max(magnitude(u.z), magnitude(u.w)));
}

// DELTA: 0 none, 1 binary16, 2 float32. A vector is four values. WIDE: blocks of more than kNarrowThreads, held to registers that let two
// of them onto an SM (12288 float32 values a row, 4096 rows: 63 us with one, 46 with two); narrow blocks are faster with all they ask for. (At 40
// registers the float32 delta's form without values spills 16 bytes; no other does.)
template <int DELTA, bool WIDE, bool VALUES>
__global__ void __launch_bounds__(WIDE ? kMaxThreads : kNarrowThreads, WIDE ? 2 : 1) rms_norm_s8_kernel(const RowsParams p) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const std::size_t row = blockIdx.x;
    const unsigned vecs = static_cast<unsigned>(p.cols / 4);
    float4* const xr = reinterpret_cast<float4*>(const_cast<float*>(static_cast<const float*>(p.x)) + row * p.ld_x);
    const float4* const gain = reinterpret_cast<const float4*>(p.w);
    const float4* const smooth = reinterpret_cast<const float4*>(p.col_scale);
    const auto added = [&](unsigned c) {
        float4 v = load_once_f32(xr + c);
        if constexpr (DELTA != 0) {
            float4 d;
            if constexpr (DELTA == 1) {
                const uint2 raw = reinterpret_cast<const uint2*>(static_cast<const __half*>(p.delta) + row * p.ld_delta)[c];
                const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
                d = make_float4(lo.x, lo.y, hi.x, hi.y);
            } else {
                d = load_once_f32(reinterpret_cast<const float4*>(static_cast<const float*>(p.delta) + row * p.ld_delta) + c);
            }
            v = make_float4(__fadd_rn(v.x, d.x), __fadd_rn(v.y, d.y), __fadd_rn(v.z, d.z), __fadd_rn(v.w, d.w));
        }
        return v;
    };
    const auto gained = [&](const float4& v, unsigned c) {
        float4 g = gain[c];
        g = make_float4(__fadd_rn(1.0f, g.x), __fadd_rn(1.0f, g.y), __fadd_rn(1.0f, g.z), __fadd_rn(1.0f, g.w));
        if (smooth != nullptr) g = product(g, smooth[c]);
        return product(v, g);
    };

    float4 held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const unsigned c = threadIdx.x + blockDim.x * i;
        held[i] = c < vecs ? added(c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float sum = 0.0f;
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const unsigned c = threadIdx.x + blockDim.x * i;
        if (c < vecs) {
            if constexpr (DELTA != 0) xr[c] = held[i];
            sum = square_into(sum, held[i]);
            held[i] = gained(held[i], c);
            top = largest_of(top, held[i]);
        }
    }
    for (unsigned c = threadIdx.x + blockDim.x * kHeld; c < vecs; c += blockDim.x) {
        const float4 v = added(c);
        if constexpr (DELTA != 0) xr[c] = v;
        sum = square_into(sum, v);
        top = largest_of(top, gained(v, c));
    }
    reduce_row<true>(sum, top);
    const RowScale s = row_scale<true>(sum, top, p);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const unsigned c = threadIdx.x + blockDim.x * i;
        if (c < vecs) store_vector<VALUES>(p, row, c, {held[i].x, held[i].y, held[i].z, held[i].w}, s);
    }
    for (unsigned c = threadIdx.x + blockDim.x * kHeld; c < vecs; c += blockDim.x) {
        const float4 u = gained(xr[c], c);  // this thread's own write, where there was one
        store_vector<VALUES>(p, row, c, {u.x, u.y, u.z, u.w}, s);
    }
    if (threadIdx.x == 0) p.scales[row] = s.scale;
}

// A vector of a row to quantise is 16 bytes of x, eight binary16 values or four float32 ones: its values, scaled.
template <bool HALF>
__device__ __forceinline__ void row_values(const uint4& raw, const float4* smooth, unsigned c, float (&v)[HALF ? 8 : 4]) {
    if constexpr (HALF) {
        widen(raw, v);
    } else {
        v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y), v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
    }
    if (smooth == nullptr) return;
#pragma unroll
    for (int h = 0; h < (HALF ? 2 : 1); ++h) {
        const float4 m = smooth[c * (HALF ? 2 : 1) + h];
        v[4 * h] = __fmul_rn(v[4 * h], m.x), v[4 * h + 1] = __fmul_rn(v[4 * h + 1], m.y);
        v[4 * h + 2] = __fmul_rn(v[4 * h + 2], m.z), v[4 * h + 3] = __fmul_rn(v[4 * h + 3], m.w);
    }
}
// Quantisation alone, a block to a row; the vectors are kept as they came.
template <bool HALF, bool WIDE, bool VALUES>
__global__ void __launch_bounds__(WIDE ? kMaxThreads : kNarrowThreads, WIDE ? 2 : 1) quantize_tokens_s8_kernel(const RowsParams p) {
    constexpr int kValues = HALF ? 8 : 4;
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const std::size_t row = blockIdx.x;
    const unsigned vecs = static_cast<unsigned>(p.cols / kValues);
    const uint4* const xr = reinterpret_cast<const uint4*>(static_cast<const char*>(p.x) + row * p.ld_x * (HALF ? 2 : 4));
    const float4* const smooth = reinterpret_cast<const float4*>(p.col_scale);
    const auto largest = [&](unsigned top, const uint4& raw, unsigned c) {
        float v[kValues];
        row_values<HALF>(raw, smooth, c, v);
#pragma unroll
        for (int j = 0; j < kValues; ++j) top = max(top, magnitude(v[j]));
        return top;
    };
    uint4 held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const unsigned c = threadIdx.x + blockDim.x * i;
        if (c < vecs) held[i] = load_once(xr + c);
    }
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const unsigned c = threadIdx.x + blockDim.x * i;
        if (c < vecs) top = largest(top, held[i], c);
    }
    for (unsigned c = threadIdx.x + blockDim.x * kHeld; c < vecs; c += blockDim.x) top = largest(top, xr[c], c);
    float none = 0.0f;
    reduce_row<false>(none, top);
    const RowScale s = row_scale<false>(0.0f, top, p);
    const auto store = [&](const uint4& raw, unsigned c) {
        float v[kValues];
        row_values<HALF>(raw, smooth, c, v);
        store_vector<VALUES>(p, row, c, v, s);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const unsigned c = threadIdx.x + blockDim.x * i;
        if (c < vecs) store(held[i], c);
    }
    for (unsigned c = threadIdx.x + blockDim.x * kHeld; c < vecs; c += blockDim.x) store(xr[c], c);
    if (threadIdx.x == 0) p.scales[row] = s.scale;
}

// Any alignment and any length, a value at a time; the same arithmetic in the same order. A thread reads back only what it wrote itself.
template <bool NORM, bool HALF, int DELTA>
__global__ void __launch_bounds__(kMaxThreads) rows_s8_any_kernel(const RowsParams p) {
    ptx::grid_launch_dependents();
    ptx::grid_dependency_wait();
    const std::size_t row = blockIdx.x;
    const auto fetch = [&](std::size_t c) {
        if constexpr (HALF)
            return __half2float(static_cast<const __half*>(p.x)[row * p.ld_x + c]);
        else
            return static_cast<const float*>(p.x)[row * p.ld_x + c];
    };
    const auto gained = [&](float v, std::size_t c) {
        if constexpr (NORM) {
            const float g = __fadd_rn(1.0f, p.w[c]);
            return __fmul_rn(v, p.col_scale != nullptr ? __fmul_rn(g, p.col_scale[c]) : g);
        }
        return p.col_scale != nullptr ? __fmul_rn(v, p.col_scale[c]) : v;
    };
    float sum = 0.0f;
    unsigned top = 0;
    for (std::size_t first = 4 * static_cast<std::size_t>(threadIdx.x); first < p.cols; first += 4 * static_cast<std::size_t>(blockDim.x)) {
        const std::size_t end = first + 4 < p.cols ? first + 4 : p.cols;
        for (std::size_t c = first; c < end; ++c) {
            float v = fetch(c);
            if constexpr (DELTA != 0) {
                const std::size_t at = row * p.ld_delta + c;
                v = __fadd_rn(v, DELTA == 1 ? __half2float(static_cast<const __half*>(p.delta)[at]) : static_cast<const float*>(p.delta)[at]);
                const_cast<float*>(static_cast<const float*>(p.x))[row * p.ld_x + c] = v;
            }
            if constexpr (NORM) sum = __fmaf_rn(v, v, sum);
            top = max(top, magnitude(gained(v, c)));
        }
    }
    reduce_row<NORM>(sum, top);
    const RowScale s = row_scale<NORM>(sum, top, p);
    for (std::size_t first = 4 * static_cast<std::size_t>(threadIdx.x); first < p.cols; first += 4 * static_cast<std::size_t>(blockDim.x)) {
        const std::size_t end = first + 4 < p.cols ? first + 4 : p.cols;
        for (std::size_t c = first; c < end; ++c) {
            const float r = s.finite ? rounded(gained(fetch(c), c), s) : kRound;
            p.q[row * p.ld_q + c] = static_cast<std::int8_t>(byte_of(r));
            if (p.values != nullptr) p.values[row * p.ld_values + c] = value_of(r, s);
        }
    }
    if (threadIdx.x == 0) p.scales[row] = s.scale;
}

bool aligned(const void* ptr, std::size_t bytes) { return reinterpret_cast<std::uintptr_t>(ptr) % bytes == 0; }

// As few threads as hold the row in kHeld vectors each, in whole warps.
unsigned threads_for(std::size_t vecs) {
    const std::size_t want = ((vecs + kHeld - 1) / kHeld + 31) / 32 * 32;
    return want > kMaxThreads ? kMaxThreads : static_cast<unsigned>(want);
}

using RowsKernel = void (*)(RowsParams);
template <int DELTA>
RowsKernel norm_kernel(unsigned threads, const void* values) {
    if (threads > kNarrowThreads) return values != nullptr ? rms_norm_s8_kernel<DELTA, true, true> : rms_norm_s8_kernel<DELTA, true, false>;
    return values != nullptr ? rms_norm_s8_kernel<DELTA, false, true> : rms_norm_s8_kernel<DELTA, false, false>;
}
template <bool HALF>
RowsKernel quantise_kernel(unsigned threads, const void* values) {
    if (threads > kNarrowThreads) return values != nullptr ? quantize_tokens_s8_kernel<HALF, true, true> : quantize_tokens_s8_kernel<HALF, true, false>;
    return values != nullptr ? quantize_tokens_s8_kernel<HALF, false, true> : quantize_tokens_s8_kernel<HALF, false, false>;
}

void check_rows(const char* who, std::size_t rows, std::size_t cols, std::size_t ld_x, std::size_t ld_q, const void* values, std::size_t ld_values) {
    if (cols == 0 || ld_x < cols || ld_q < cols || (values != nullptr && ld_values < cols)) throw std::invalid_argument(std::string(who) + ": a row has at least one value and the strides hold a row");
    if (rows > 0x7FFFFFFFu || cols > 0x7FFFFFFFu) throw std::invalid_argument(std::string(who) + ": dimension beyond 2^31");
}

}  // namespace

bool norm_s8_takes_eps(float eps) { return eps >= 1.0e-30f && std::isfinite(eps); }

void launch_rms_norm_s8(const Context& ctx, float* x, std::size_t ld_x, const void* delta, std::size_t ld_delta, bool delta_half, const float* w, const float* col_scale,
                        std::int8_t* q, std::size_t ld_q, float* scales, void* values, std::size_t ld_values, std::size_t rows, std::size_t cols, float eps, cudaStream_t stream) {
    check_rows("launch_rms_norm_s8", rows, cols, ld_x, ld_q, values, ld_values);
    if (delta != nullptr && ld_delta < cols) throw std::invalid_argument("launch_rms_norm_s8: the stride of delta does not hold a row");
    if (!norm_s8_takes_eps(eps)) throw std::invalid_argument("launch_rms_norm_s8: eps must be a positive number (1e-30 at least)");
    if (rows == 0) return;
    if (x == nullptr || w == nullptr || q == nullptr || scales == nullptr) throw std::invalid_argument("launch_rms_norm_s8: null pointer");
    if (!aligned(x, 4) || !aligned(w, 4) || !aligned(scales, 4) || !aligned(col_scale, 4) || !aligned(delta, delta_half ? 2 : 4) || !aligned(values, 2))
        throw std::invalid_argument("launch_rms_norm_s8: a pointer is not aligned to its values");
    check(cudaSetDevice(ctx.device), "cudaSetDevice");
    const RowsParams p{x, ld_x, delta, ld_delta, w, col_scale, q, ld_q, scales, static_cast<__half*>(values), ld_values, cols, eps};
    const unsigned kind = delta == nullptr ? 0u : delta_half ? 1u : 2u;
    const bool vectors = cols % 4 == 0 && ld_x % 4 == 0 && ld_q % 4 == 0 && aligned(x, 16) && aligned(w, 16) && aligned(q, 4) &&
                         (col_scale == nullptr || aligned(col_scale, 16)) && (kind == 0 || (ld_delta % 4 == 0 && aligned(delta, delta_half ? 8 : 16))) && (values == nullptr || (ld_values % 4 == 0 && aligned(values, 8)));
    const dim3 grid(static_cast<unsigned>(rows));
    if (vectors) {
        const unsigned threads = threads_for(cols / 4);
        launch_kernel(kind == 0 ? norm_kernel<0>(threads, values) : kind == 1 ? norm_kernel<1>(threads, values) : norm_kernel<2>(threads, values), grid,
                      dim3(threads), 0, stream, "rms_norm_s8_kernel launch", p);
    } else {
        const auto kernel = kind == 0 ? rows_s8_any_kernel<true, false, 0> : kind == 1 ? rows_s8_any_kernel<true, false, 1> : rows_s8_any_kernel<true, false, 2>;
        launch_kernel(kernel, grid, dim3(threads_for((cols + 3) / 4)), 0, stream, "rows_s8_any_kernel launch", p);
    }
    count_launch();
}

void launch_quantize_tokens_s8(const Context& ctx, const void* x, std::size_t ld_x, bool x_half, const float* col_scale, std::int8_t* q, std::size_t ld_q, float* scales, void* values, std::size_t ld_values,
                               std::size_t rows, std::size_t cols, cudaStream_t stream) {
    check_rows("launch_quantize_tokens_s8", rows, cols, ld_x, ld_q, values, ld_values);
    if (rows == 0) return;
    if (x == nullptr || q == nullptr || scales == nullptr) throw std::invalid_argument("launch_quantize_tokens_s8: null pointer");
    if (!aligned(x, x_half ? 2 : 4) || !aligned(scales, 4) || !aligned(col_scale, 4) || !aligned(values, 2))
        throw std::invalid_argument("launch_quantize_tokens_s8: a pointer is not aligned to its values");
    check(cudaSetDevice(ctx.device), "cudaSetDevice");
    const RowsParams p{x, ld_x, nullptr, 0, nullptr, col_scale, q, ld_q, scales, static_cast<__half*>(values), ld_values, cols, 0.0f};
    const std::size_t per_vec = x_half ? 8 : 4;
    const bool vectors = cols % per_vec == 0 && ld_x % per_vec == 0 && ld_q % per_vec == 0 && aligned(x, 16) && aligned(q, per_vec) &&
                         (col_scale == nullptr || aligned(col_scale, 16)) && (values == nullptr || (ld_values % per_vec == 0 && aligned(values, 2 * per_vec)));
    const dim3 grid(static_cast<unsigned>(rows));
    if (vectors) {
        const unsigned threads = threads_for(cols / per_vec);
        launch_kernel(x_half ? quantise_kernel<true>(threads, values) : quantise_kernel<false>(threads, values), grid, dim3(threads), 0, stream,
                      "quantize_tokens_s8_kernel launch", p);
    } else {
        const auto kernel = x_half ? rows_s8_any_kernel<false, true, 0> : rows_s8_any_kernel<false, false, 0>;
        launch_kernel(kernel, grid, dim3(threads_for((cols + 3) / 4)), 0, stream, "rows_s8_any_kernel launch", p);
    }
    count_launch();
}

}  // namespace sepal::b200
