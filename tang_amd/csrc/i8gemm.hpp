// Products of 8-bit integers with a scale for each token and each channel.
//
//   s_i = f32(max_k |x_ik| / 127), q_ik = x_ik / s_i to the nearest integer (ties to even)
//   y_ij = (sum_k q_ik w_jk) s_i t_j + b_j
//
// w are the q8 weights with one scale a row (th_qweight in common.hpp), whose tiles
// of 16 rows x 64 k are, lane by lane, an operand of the 16x16x64 i8 MFMA.  q lies
// the same way (a load of 1 KiB then is eight lines instead of pieces of sixteen:
// 64 rows, 4096 x 4096 12.0 -> 8.5 us), but for a last block of h < 16 rows, which
// takes their bytes alone: value (i, k) is at
//   (i - i % 16) Kp + (k - k % 16) h + i % 16 * 16 + k % 16,
// Kp = K rounded up to 64.  What lies behind K meets zero weights.
#pragma once

#include "common.hpp"

namespace th {

// Sums of K products of two int8 (at most 2^14 each) stay in 32 bits below this.
constexpr size_t I8_MAX_K = ((size_t)1 << 17) - 1;
// Rows of a weight: 2^23 tiles of 16 by 512 threads would be the 2^32 that a launch stays below.
constexpr size_t I8_MAX_ROWS = ((size_t)1 << 27) - 16;

// Where results go: (sum s_i) t_j + b_j, so formed that no order of the scales
// leaves f32's range on the way (i8kernels.hpp), and rounded to the output's type.
struct I8Out {
    void* y;
    const float *xs, *ws, *bias;  // [M], [N], [N] or null
    th_dtype dt;                  // of y
    int N;
};

// The kernel of a product (i8gemm.hip): of up to 64 rows, by tiles of 16 channels and of 16 rows that a workgroup has; of more, by
// the tile's rows and channels.  At most i8_rows_at_once(n) rows go to a launch.
enum class I8Form { ROWS_1X1, ROWS_1X2, ROWS_2X2, ROWS_1X4, ROWS_2X4, ROWS_3X4, TILE_64X64, TILE_64X128_TWO, TILE_64X128, TILE_128X128, TILE_128X256, TILE_256X256 };
I8Form i8_form(size_t m, size_t n, size_t k, size_t cus);
size_t i8_rows_at_once(size_t n);

// whole: the last block too has 16 rows, zeros (and scales of zero) behind the m.
void launch_quantize_rows(const void* x, th_dtype xdt, size_t m, size_t K, int8_t* q, float* scale, bool whole, hipStream_t s);
void launch_q8_pack(const int8_t* q, const float* scale, const th_qweight* w, hipStream_t s);
void launch_i8_linear(th_device* dev, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m);

}  // namespace th
