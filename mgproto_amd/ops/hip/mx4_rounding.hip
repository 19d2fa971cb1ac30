// Products whose rows are rounded on the way: y = Q(x) W^T + bias for many rows
// and few columns, where the time is x's way from memory.
//
// A block of 64 rows takes all columns it can (up to 256), so that x is read and
// rounded once for each 256 of them. Two buffers of 128 elements: while the
// matrix cores work on one, the weights' codes go into the other past the
// registers, and the next rows of x come into registers, are rounded there
// (four lanes share a block, two lane exchanges for its maximum) and written as
// codes. One barrier a buffer.
//
// Bound by x's way from memory: 62720x1024->256 takes 34 us where the caches hold x
// (4.8 TB/s), 39 where not, 250880x256->64 27 (6.0). Two blocks and more share a
// unit, so that one reads while another starts or writes: tiles of 128 rows and 256
// elements, one on a unit, took 39 and 38; four waves for 256 columns instead of
// eight 37 and 42 (62720x333->200 24 and 28 for 20 and 24). x two steps ahead: 36,
// 62720x512->128 18 for 16.

#include <hip/hip_runtime.h>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

template <int DT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN)
void rounding_kernel(const typename Elem<DT>::T* __restrict__ x, long M, int K,
                     int steps, long ldx, const uint8_t* __restrict__ wc,
                     const uint8_t* __restrict__ ws, long N,
                     const void* __restrict__ bias, int bias_dt,
                     typename Elem<DT>::T* __restrict__ y, int nt, int total) {
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int W = DT == F32 ? 2 : 1;
    constexpr int UNITS = BM * 16 / THREADS;     // of 8 elements, 16 a row
    constexpr int CALLS = BN / 16;               // copies of a step's codes
    // codes of a step; x's scale bytes, 4 a row; W's as stored, of four steps
    __shared__ __attribute__((aligned(16))) uint8_t xl[2][BM * 64];
    __shared__ __attribute__((aligned(16))) uint8_t wl[2][BN * 64];
    __shared__ __attribute__((aligned(16))) uint8_t xsl[2][BM * 4];
    __shared__ __attribute__((aligned(16))) uint8_t wsl[2][BN * 16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int wm = (wave / WN) * (FM * 16), wn = (wave % WN) * (FN * 16);

    // Blocks go round the 8 dies; a die has a run of tiles, the columns of the
    // same rows one after the other, so that x comes from its L2 again.
    const int xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
    const int t = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
    const long m0 = (long)(t / nt) * BM, n0 = (long)(t % nt) * BN;
    const int lastw = (int)min((long)BN, N - n0) - 1;
    const int lastx = (int)min((long)BM, M - m0) - 1;

    auto send_w = [&](int k, int buf) {
        #pragma unroll
        for (int q = 0; q < CALLS / WAVES; ++q) {
            const int c = q * WAVES + wave, r = c * 16 + (lane >> 2);
            copy16_to_lds(wc + ((size_t)k * N + n0) * 64,
                          min(r, lastw) * 64 + ((lane & 3) ^ w_key<FN>(r)) * 16,
                          lds_address(wl[buf]) + c * 1024);
        }
        if ((k & 3) == 0 && wave < BN / 64) {    // four steps' scales
            const int r = wave * 64 + lane;
            copy16_to_lds(ws + ((size_t)(k >> 2) * N + n0) * 16,
                          min(r, lastw) * 16,
                          lds_address(wsl[k >> 2 & 1]) + wave * 1024);
        }
    };
    u32x4 raw[UNITS][W];
    const typename Elem<DT>::T* x0 = x + m0 * ldx;
    auto load_x = [&](int k) {
        #pragma unroll
        for (int q = 0; q < UNITS; ++q) {
            const int u = q * THREADS + tid, r = u >> 4;
            const int at = k * 128 + (u & 15) * 8;
            const typename Elem<DT>::T* p = x0 + min(r, lastx) * ldx + at;
            if (at + 8 <= K) load8<DT>(p, raw[q]);
            else load8_tail<DT>(p, K - at, raw[q]);
        }
    };
    auto store_x = [&](int buf) {
        #pragma unroll
        for (int q = 0; q < UNITS; ++q) {
            const int u = q * THREADS + tid, r = u >> 4, c8 = u & 15, b = c8 >> 2;
            const unsigned byte = scale_byte<DT>(quad_max(absmax_bits<DT>(raw[q], W)));
            const unsigned c = codes8<DT>(raw[q], scale_f32(byte));
            *reinterpret_cast<unsigned*>(
                xl[buf] + r * 64 + ((b ^ x_key(r)) << 4) + (c8 & 3) * 4) = c;
            if ((c8 & 3) == 0) xsl[buf][r * 4 + b] = (uint8_t)byte;
        }
    };

    f32x4 acc[FM][FN];
    #pragma unroll
    for (int i = 0; i < FM; ++i)
        #pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

    const int xr = wm + r16, wr = wn + (r16 >> 2) * (4 * FN) + (r16 & 3);
    const int xp = xr * 64 + ((g ^ x_key(xr)) << 4);
    const int wp = wr * 64 + ((g ^ w_key<FN>(wr)) << 4);
    int wb[FN];                          // scales of this step and up to 3 more
    auto compute = [&](int k, int buf) {
        int xb[FM];
        i32x4 w[FN];
        if ((k & 3) == 0) {
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                wb[j] = *reinterpret_cast<const int*>(
                    wsl[k >> 2 & 1] + (wr + j * 4) * 16 + g * 4);
        } else {
            #pragma unroll
            for (int j = 0; j < FN; ++j) wb[j] = (unsigned)wb[j] >> 8;
        }
        #pragma unroll
        for (int i = 0; i < FM; ++i) xb[i] = xsl[buf][(xr + i * 16) * 4 + g];
        #pragma unroll
        for (int j = 0; j < FN; ++j)
            w[j] = *reinterpret_cast<const i32x4*>(wl[buf] + wp + j * 256);
        #pragma unroll
        for (int i = 0; i < FM; ++i) {
            const i32x4 a = *reinterpret_cast<const i32x4*>(xl[buf] + xp + i * 1024);
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    wide(w[j]), wide(a), acc[i][j], 4, 4, 0, wb[j], 0, xb[i]);
        }
    };
    if (steps) {
        send_w(0, 0);
        load_x(0);
        store_x(0);
    }
    for (int k = 0; k < steps; ++k) {
        // the buffer's bytes have arrived, and no wave reads the other one any
        // more
        wait_copies<0>();
        __syncthreads();
        if (k + 1 < steps) {
            send_w(k + 1, (k + 1) & 1);
            load_x(k + 1);
        }
        compute(k, k & 1);
        if (k + 1 < steps) store_x((k + 1) & 1);
    }

    const long n = n0 + wn + g * (4 * FN);
    float b[4 * FN];
    load_bias<FN>(b, bias, bias_dt, n, N);
    store_rows<DT, FM, FN>(acc, y, M, N, m0 + wm + r16, n, b);
}

template <int DT, int BM, int BN, int WM, int WN>
void launch_rounding(const void* x, long M, long K, long ldx,
                     const uint8_t* wc, const uint8_t* ws, long N,
                     const void* bias, int bias_dt, void* y,
                     hipStream_t stream) {
    using T = typename Elem<DT>::T;
    const int mt = (int)((M + BM - 1) / BM), nt = (int)((N + BN - 1) / BN);
    hipLaunchKernelGGL((rounding_kernel<DT, BM, BN, WM, WN>),
                       dim3((unsigned)(mt * nt)), dim3(64 * WM * WN), 0, stream,
                       (const T*)x, M, (int)K, (int)steps_of(K), ldx, wc, ws, N,
                       bias, bias_dt, (T*)y, nt, mt * nt);
}

}  // namespace

void rounding(const void* x, int dt, long M, long K, long ldx,
              const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
              int bias_dt, void* y, hipStream_t stream) {
    #define MX4_T(DT, BN, WM, WN) \
        launch_rounding<DT, 64, BN, WM, WN>(x, M, K, ldx, wc, ws, N, bias, \
                                            bias_dt, y, stream)
    #define MX4_D(BN, WM, WN) do { \
        if (dt == F32) MX4_T(F32, BN, WM, WN); \
        else if (dt == BF16) MX4_T(BF16, BN, WM, WN); \
        else MX4_T(F16, BN, WM, WN); } while (0)
    if (N > 128) MX4_D(256, 2, 4);
    else if (N > 64) MX4_D(128, 2, 2);
    else MX4_D(64, 4, 1);
    #undef MX4_D
    #undef MX4_T
}

}  // namespace mx4
