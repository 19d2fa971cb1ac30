// Pieces that the products of 4-bit rows share.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx4_common.h"

namespace mx4 {

static __device__ __forceinline__ i32x8 wide(i32x4 v) {
    return (i32x8){v.x, v.y, v.z, v.w, 0, 0, 0, 0};
}

static __device__ __forceinline__ float load_any(const void* p, int dt, long i) {
    if (dt == F32) return reinterpret_cast<const float*>(p)[i];
    if (dt == BF16) return (float)reinterpret_cast<const __bf16*>(p)[i];
    return (float)reinterpret_cast<const _Float16*>(p)[i];
}

// maximum over the four lanes of a quad
static __device__ __forceinline__ unsigned quad_max(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));
    return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));
}

// Rows m, m + 16, ... of y from column n on: 4*FN consecutive columns a lane.
// Pieces of 16 bytes where rows start on them, single elements elsewhere.
template <int OT, int FM, int FN>
static __device__ __forceinline__ void store_rows(
        const f32x4 (&acc)[FM][FN], typename Elem<OT>::T* y, long M, long N,
        long m, long n, const void* bias, int bias_dt) {
    using T = typename Elem<OT>::T;
    constexpr int PER = OT == F32 ? 1 : (FN % 2 ? 1 : 2);   // tiles a piece
    constexpr int W = 4 * PER;                              // columns a piece
    const bool vec = N % W == 0;
    #pragma unroll
    for (int j = 0; j < FN; j += PER) {
        const long c = n + j * 4;
        float b[W];
        #pragma unroll
        for (int r = 0; r < W; ++r)
            b[r] = bias && c + r < N ? load_any(bias, bias_dt, c + r) : 0.f;
        #pragma unroll
        for (int i = 0; i < FM; ++i) {
            const long row = m + i * 16;
            if (row >= M || c >= N) continue;
            T* q = y + row * N + c;
            union { T v[W]; u32x2 h[W * sizeof(T) / 8]; } o;
            #pragma unroll
            for (int r = 0; r < W; ++r)
                o.v[r] = from_f32<OT>(acc[i][j + r / 4][r % 4] + b[r]);
            if (vec) {
                if constexpr (W * sizeof(T) == 16)
                    *reinterpret_cast<u32x4*>(q) =
                        (u32x4){o.h[0].x, o.h[0].y, o.h[1].x, o.h[1].y};
                else
                    *reinterpret_cast<u32x2*>(q) = o.h[0];
            } else {
                #pragma unroll
                for (int r = 0; r < W; ++r)
                    if (c + r < N) q[r] = o.v[r];
            }
        }
    }
}

// mx4_tiled.hip
void tiled_q(const uint8_t* xc, const uint8_t* xs, long M, long K,
             const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
             int bias_dt, void* y, int dt, bool large, hipStream_t stream);
void tiled(const void* x, int dt, bool vec, long M, long K, long ldx,
           const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
           int bias_dt, void* y, hipStream_t stream);

}  // namespace mx4
