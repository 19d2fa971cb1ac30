// Pieces that the products of 4-bit rows share.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "mx4_common.h"

namespace mx4 {

static __device__ __forceinline__ i32x8 wide(i32x4 v) {
    return (i32x8){v.x, v.y, v.z, v.w, 0, 0, 0, 0};
}

// The values of 8 codes under one scale byte. (Byte 255 becomes an infinite
// scale here, which the conversion takes for not a number, as it should.)
static __device__ __forceinline__ void values8(unsigned c, unsigned byte,
                                               float (&f)[8]) {
    const float s = scale_f32(byte);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
    const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    f[4] = d.x; f[5] = d.y; f[6] = e.x; f[7] = e.y;
}

// 16 bytes a lane from memory into LDS, past the registers: lane i's, from
// base + off, go to l + 16 i; base and l are the same in the wave. In assembly,
// because the compiler would wait for every such copy before the next read of
// LDS, whichever bytes that reads: waiting is the caller's, by wait_copies() and
// a barrier. No register is written. The pause covers a base that a vector
// instruction wrote just before.
static __device__ __forceinline__ unsigned lds_address(const void* l) {
    return (unsigned)(uintptr_t)l;
}
static __device__ __forceinline__ void copy16_to_lds(const void* base,
                                                     unsigned off, unsigned l) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\t"
                 "global_load_lds_dwordx4 %0, %1"
                 :: "v"(off), "s"(base), "s"(l) : "memory", "m0");
}
// until at most N of this wave's memory instructions are under way (they end
// in their order), and its reads of LDS are over
template <int N> static __device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
}

// In LDS a step's codes are rows of 64 bytes, four pieces of 16; piece g of row
// r lies at g ^ key(r). A read takes 16 bytes a lane, lane group g piece g of 16
// rows, and is served in four turns: lanes 0-3, 12-15 and 20-27 together, 4-11,
// 16-19 and 28-31 together, and so on. These keys put a turn's 16 pieces on 16
// different places of the 256 bytes that the banks give at once (measured: 4
// cycles a read, 8 without a key).
// rows of x are read 16 consecutive ones at a time
static __device__ __forceinline__ int x_key(int r) { return r >> 1 & 3; }
// rows of W in four runs of four, 4*FN apart
template <int FN> static __device__ __forceinline__ int w_key(int r) {
    return r / (4 * FN) & 2;
}

// maximum over the four lanes of a quad
static __device__ __forceinline__ unsigned quad_max(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));
    return max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));
}

// 4*FN values of the bias from column n on, 0 where there is none
template <int FN>
static __device__ __forceinline__ void load_bias(float (&b)[4 * FN],
                                                 const void* bias, int dt,
                                                 long n, long N) {
    #pragma unroll
    for (int i = 0; i < 4 * FN; ++i) b[i] = 0.f;
    if (!bias) return;
    if (dt == F32) {
        const float* p = reinterpret_cast<const float*>(bias);
        #pragma unroll
        for (int i = 0; i < 4 * FN; ++i) b[i] = p[min(n + i, N - 1)];
        // (waited for here, not in every step of the loop that comes next)
        #pragma unroll
        for (int i = 0; i < 4 * FN; ++i) asm volatile("" : "+v"(b[i]));
    } else {
        const unsigned short* p = reinterpret_cast<const unsigned short*>(bias);
        unsigned short u[4 * FN];
        #pragma unroll
        for (int i = 0; i < 4 * FN; ++i) u[i] = p[min(n + i, N - 1)];
        #pragma unroll
        for (int i = 0; i < 4 * FN; ++i)
            b[i] = dt == BF16 ? __uint_as_float((unsigned)u[i] << 16)
                              : (float)__builtin_bit_cast(_Float16, u[i]);
    }
}

// Pieces of 16 bytes in lane groups of 16: piece i of group g becomes piece g of
// "row" i, so that a store's four groups write 64 bytes in one run instead of 16
// at a distance each: 62720x256->1024 from 4-bit rows 30 -> 28 us, 15680x512->2048
// 22.3 -> 20.7.
template <int P>
static __device__ __forceinline__ void gather_pieces(u32x4 (&p)[P]) {
    auto swap16 = [](u32x4& a, u32x4& b) {   // odd groups of a, even ones of b
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto r = __builtin_amdgcn_permlane16_swap(a[i], b[i], false, false);
            a[i] = r[0], b[i] = r[1];
        }
    };
    auto swap32 = [](u32x4& a, u32x4& b) {   // upper half of a, lower of b
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap(a[i], b[i], false, false);
            a[i] = r[0], b[i] = r[1];
        }
    };
    if constexpr (P == 2) {
        swap16(p[0], p[1]);
        swap32(p[0], p[1]);
    } else if constexpr (P == 4) {
        swap16(p[0], p[1]);
        swap16(p[2], p[3]);
        swap32(p[0], p[2]);
        swap32(p[1], p[3]);
    }
}

// Rows m, m + 16, ... of y from column n on: 4*FN consecutive columns a lane,
// in pieces of 16 bytes, wherever a row starts; single elements at its end.
template <int OT, int FM, int FN>
static __device__ __forceinline__ void store_rows(
        const f32x4 (&acc)[FM][FN], typename Elem<OT>::T* y, long M, long N,
        long m, long n, const float (&b)[4 * FN]) {
    using T = typename Elem<OT>::T;
    constexpr int PER = OT == F32 ? 1 : (FN % 2 ? 1 : 2);   // tiles a piece
    constexpr int W = 4 * PER;                              // columns a piece
    constexpr int P = FN / PER;                             // pieces a lane
    constexpr bool TURN = W * sizeof(T) == 16 && (P == 2 || P == 4);
    const int g = (threadIdx.x & 63) >> 4;
    // the first piece's column, and the way to the next
    const long n0 = TURN ? n - g * (4 * FN) + g * W : n;
    constexpr int step = TURN ? 4 * W : W;
    #pragma unroll
    for (int i = 0; i < FM; ++i) {
        Piece<T, W> o[P];
        #pragma unroll
        for (int j = 0; j < FN; ++j)
            #pragma unroll
            for (int r = 0; r < 4; ++r)
                o[j / PER].v[j % PER * 4 + r] =
                    from_f32<OT>(acc[i][j][r] + b[j * 4 + r]);
        if constexpr (TURN) {
            u32x4 u[P];
            #pragma unroll
            for (int p = 0; p < P; ++p) u[p] = o[p].u[0];
            gather_pieces<P>(u);
            #pragma unroll
            for (int p = 0; p < P; ++p) o[p].u[0] = u[p];
        }
        const long row = m + i * 16;
        if (row >= M) continue;
        #pragma unroll
        for (int p = 0; p < P; ++p) {
            const long c = n0 + p * step;
            store_piece(y + row * N + c, o[p], N - c);
        }
    }
}

// mx4_tiles.hip
void tiles(const uint8_t* xc, const uint8_t* xs, long M, long K,
           const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
           int bias_dt, void* y, int dt, bool large, hipStream_t stream);
// mx4_rounding.hip
void rounding(const void* x, int dt, long M, long K, long ldx,
              const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
              int bias_dt, void* y, hipStream_t stream);

}  // namespace mx4
