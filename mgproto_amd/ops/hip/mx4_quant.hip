// Rows to MX4 blocks and back. See mx4_common.h for the format.
//
// Bound by memory: 2 (or 4) bytes in and 0.53 out an element, the reverse for
// reading back. Four lanes share a block, 8 elements each, so that a wave
// reads 1 KB (16-bit) or 2 KB (fp32) in one piece and writes 256 bytes of
// codes in one; the block's maximum goes over the four lanes by two shuffles.

#include <hip/hip_runtime.h>

#include "mx4_common.h"

namespace mx4 {
namespace {

template <int DT, bool VEC>
__global__ __launch_bounds__(256)
void quantize_kernel(const typename Elem<DT>::T* __restrict__ x, long rows,
                     int K, int Kp, long ldx, unsigned* __restrict__ codes,
                     uint8_t* __restrict__ scales) {
    constexpr int W = DT == F32 ? 2 : 1;
    const int upr = Kp >> 3;                     // units of 8 in a row
    const long total = rows * upr;
    const long step = (long)gridDim.x * 256;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
        const long row = t / upr;
        const int k = (int)(t - row * upr) << 3;
        u32x4 u[W];
        const typename Elem<DT>::T* p = x + row * ldx + k;
        if (VEC && k + 8 <= K) {
            #pragma unroll
            for (int i = 0; i < W; ++i)
                u[i] = reinterpret_cast<const u32x4*>(p)[i];
        } else {
            load8_tail<DT>(p, K - k, u);
        }
        // upr is a multiple of 16 and so is the count of live lanes of a
        // wave: the four lanes of a block are live together
        unsigned m = absmax_bits<DT>(u, W);
        m = max(m, (unsigned)__shfl_xor((int)m, 1));
        m = max(m, (unsigned)__shfl_xor((int)m, 2));
        const unsigned byte = scale_byte<DT>(m);
        codes[t] = byte == 255u ? 0u : codes8<DT>(u, scale_f32(byte));
        if ((t & 3) == 0) scales[t >> 2] = (uint8_t)byte;
    }
}

template <int DT, bool VEC>
__global__ __launch_bounds__(256)
void dequantize_kernel(const unsigned* __restrict__ codes,
                       const uint8_t* __restrict__ scales, long rows, int K,
                       int Kp, typename Elem<DT>::T* __restrict__ out) {
    using T = typename Elem<DT>::T;
    const int upr = (K + 7) >> 3;
    const long total = rows * upr;
    const long step = (long)gridDim.x * 256;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
        const long row = t / upr;
        const int k = (int)(t - row * upr) << 3;
        const unsigned c = codes[row * (Kp >> 3) + (k >> 3)];
        const unsigned byte = scales[row * (Kp >> 5) + (k >> 5)];
        const float s = byte == 255u ? 1.f : scale_f32(byte);
        f32x2 f[4];
        f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
        f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
        f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
        f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
        union { T v[8]; u32x4 u[sizeof(T) / 2]; } o;
        #pragma unroll
        for (int i = 0; i < 8; ++i)
            o.v[i] = from_f32<DT>(byte == 255u ? __uint_as_float(0x7fc00000u)
                                               : f[i >> 1][i & 1]);
        T* q = out + row * K + k;
        if (VEC) {
            #pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                reinterpret_cast<u32x4*>(q)[i] = o.u[i];
        } else {
            for (int i = 0; i < 8 && k + i < K; ++i) q[i] = o.v[i];
        }
    }
}

unsigned grid_for(long total) {
    const long blocks = (total + 255) / 256;
    return (unsigned)(blocks < 256 * 32 ? blocks : 256 * 32);
}

}  // namespace

void quantize(const void* x, int dt, long rows, long K, long ldx,
              uint8_t* codes, uint8_t* scales, hipStream_t stream) {
    const int Kp = (int)((K + 127) / 128 * 128);
    const long total = rows * (Kp / 8);
    if (total == 0) return;
    const int es = dt == F32 ? 4 : 2;
    const bool vec = (uintptr_t)x % 16 == 0 && (ldx * es) % 16 == 0;
    #define MX4_Q(DT, V) \
        hipLaunchKernelGGL((quantize_kernel<DT, V>), dim3(grid_for(total)), \
                           dim3(256), 0, stream, \
                           (const typename Elem<DT>::T*)x, rows, (int)K, Kp, \
                           ldx, (unsigned*)codes, scales)
    if (vec) {
        if (dt == F32) MX4_Q(F32, true);
        else if (dt == BF16) MX4_Q(BF16, true);
        else MX4_Q(F16, true);
    } else {
        if (dt == F32) MX4_Q(F32, false);
        else if (dt == BF16) MX4_Q(BF16, false);
        else MX4_Q(F16, false);
    }
    #undef MX4_Q
}

void dequantize(const uint8_t* codes, const uint8_t* scales, long rows,
                long K, void* out, int dt, hipStream_t stream) {
    const int Kp = (int)((K + 127) / 128 * 128);
    const long total = rows * ((K + 7) / 8);
    if (total == 0) return;
    const bool vec = K % 8 == 0;     // fresh outputs start on 16 bytes
    #define MX4_D(DT, V) \
        hipLaunchKernelGGL((dequantize_kernel<DT, V>), dim3(grid_for(total)), \
                           dim3(256), 0, stream, (const unsigned*)codes, \
                           scales, rows, (int)K, Kp, \
                           (typename Elem<DT>::T*)out)
    if (vec) {
        if (dt == F32) MX4_D(F32, true);
        else if (dt == BF16) MX4_D(BF16, true);
        else MX4_D(F16, true);
    } else {
        if (dt == F32) MX4_D(F32, false);
        else if (dt == BF16) MX4_D(BF16, false);
        else MX4_D(F16, false);
    }
    #undef MX4_D
}

}  // namespace mx4
