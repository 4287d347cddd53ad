// Activations in 8 bits: int8 rows with one float32 scale a token, what launch_gemm_s8 (gemm_s8.hpp) multiplies.
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "context.hpp"

namespace sepal::b200 {

/// The residual's addition, the zero-centred RMSNorm and the per-token quantisation in one pass over the float32 stream:
///   x[t, :] += delta[t, :]                                    (delta null: nothing is added and x is not written)
///   v[t, c] = x[t, c] / sqrt(sum(x[t, :]^2) / cols + eps) * (1 + w[c]) * col_scale[c]        (col_scale null: 1)
///   scales[t] = max |v[t, :]| / 127,   q[t, c] = round to nearest even of v[t, c] * (127 / max |v[t, :]|)
/// values (null or binary16 [rows, ld_values]): also what the bytes stand for, binary16(q[t, c] * scales[t]).
/// delta binary16 (delta_half) or float32 [rows, cols]. In float32, the products u = x (1 + w) col_scale first and v = u over the root. A
/// row whose u is all zero gets scale 0 and zeros; a row whose x, u or v holds a NaN or an infinity, or whose squares overflow
/// float32, gets scale NaN and zeros (its products are NaN), and no other row is touched by it.
void launch_rms_norm_s8(const Context& ctx, float* x, std::size_t ld_x, const void* delta, std::size_t ld_delta, bool delta_half, const float* w, const float* col_scale,
                        std::int8_t* q, std::size_t ld_q, float* scales, void* values, std::size_t ld_values, std::size_t rows, std::size_t cols, float eps, cudaStream_t stream);

/// The eps that launch_rms_norm_s8 takes: 1e-30 or more, and finite.
bool norm_s8_takes_eps(float eps);

/// The quantisation alone, for activations that no norm makes: v = x * col_scale, then as above. x binary16 (x_half) or float32. On
/// binary16 rows of finite values the bits are those of launch_quantize_rows_s8 (with a col_scale, where the largest product is 2^-121 or more
/// or zero: below that the other's factor 127 / max overflows).
void launch_quantize_tokens_s8(const Context& ctx, const void* x, std::size_t ld_x, bool x_half, const float* col_scale, std::int8_t* q, std::size_t ld_q, float* scales, void* values, std::size_t ld_values,
                               std::size_t rows, std::size_t cols, cudaStream_t stream);

}  // namespace sepal::b200
