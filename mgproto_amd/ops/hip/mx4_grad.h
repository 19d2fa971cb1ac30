// Pieces that the gradients of the 4-bit product share.
#pragma once

#include <hip/hip_runtime.h>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {

static inline long up32(long v) { return (v + 31) / 32 * 32; }
static inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// dx = A B^T on tiles: A is `parts` matrices of M rows, read 32 elements of the
// sum at a time (64 bytes), from a + part * a_part + step * a_step + row * a_row; B
// is [steps][K][32] bf16 and serves every part. C [M, K]. tile: one of TILES, or -1
// for the one that ends first.
constexpr int TILES = 4;
void grad_input_tiles(const void* a, size_t a_step, size_t a_row, size_t a_part,
                      int parts, int steps, const void* b, long M, long K,
                      void* c, int dt, int tile, void* partial,
                      hipStream_t stream);
size_t grad_input_partial(long M, long K, long steps, int tile);

// dw = G^T X on tiles: G is `parts` matrices of M rows of N bf16, `row` elements
// apart (a multiple of 8, from 16 bytes on); X are 4-bit rows. C [N, K].
void grad_weight_tiles(const void* g, long row, size_t part, int parts, long M,
                       long N, long K, const uint8_t* xc, const uint8_t* xs,
                       void* c, int dt, void* partial, hipStream_t stream);
size_t grad_weight_partial(long M, long N, long K, int parts);

// out[i] = sum over s < S of part[s][i], in their order
void join(const float* part, int S, long n, void* out, int dt,
          hipStream_t stream);

}  // namespace mx4
