// The trunk projection on int8 activations and int8 weights (gemm_s8.cu).
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "gemm.hpp"

namespace sepal::b200 {

/// Y[t, n] = epilogue( float32(sum over k of x[t, k] * w[n, k]) * sx[t] * sw[n] ): x int8 [T, ld_x] with one float32 scale a token
/// (launch_rms_norm_s8, launch_quantize_tokens_s8), w int8 [N, ld_w] with one a row (launch_quantize_rows_s8: the matrix of launch_gemm_w8r).
/// The sums are exact 32-bit integers on the tensor cores (tcgen05.mma kind::i8), whatever the schedule: every `config` gives the same
/// bits, and a row's bits depend on nothing but the row and the weights. The two scales multiply in float32, the token's first.
///
/// `config`: -1 chooses from the shape; 512 + w (w a multiple of 32 from 32 to 256): CTA pairs, w tokens by 256 weight rows to a tile;
/// 1024 + s, 1024 + 16 + s (s 1 .. 8, at most 256 rows): the few-rows kernel, a tile's k in s parts, two CTAs to an SM (at most 128
/// rows) or one.
void launch_gemm_s8(Context& ctx, const std::int8_t* x, std::size_t ld_x, const float* sx, const std::int8_t* w, std::size_t ld_w, const float* sw, void* y,
                    std::size_t ld_y, bool y_half, std::size_t t, std::size_t n, std::size_t k, Epilogue epilogue, int config, cudaStream_t stream);

/// Values of k: a sum of 2^17 products of two bytes of -128 no longer fits 32 bits.
inline constexpr std::size_t kS8MaxK = (std::size_t{1} << 17) - 1;

}  // namespace sepal::b200
