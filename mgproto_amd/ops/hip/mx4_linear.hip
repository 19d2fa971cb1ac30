// Products of 4-bit rows: y[M,N] = Q(x)[M,K] W[N,K]^T + bias.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes, in each lane, 32 consecutive codes
// of one row and their scale byte: lane l holds row l&15, block l>>4 of a
// 128-step. That is one MX block a lane, so x can be rounded where it is
// loaded, with no word exchanged between lanes. Sums are fp32; y is rounded
// once.
//
// The weights are the first operand, so that a lane ends up with consecutive
// columns of y: output row (lane>>4)*4 + r of a tile is mapped to column
// (lane>>4)*4*FN + j*4 + r of the wave's 16*FN, 4*FN in one piece.

#include <hip/hip_runtime.h>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

constexpr int CODES = -1;     // x is held in 4 bits already

// One block of x: loaded, rounded; codes and scale byte stay in this lane.
template <int DT>
static __device__ __forceinline__ i32x4 round_block(
        const typename Elem<DT>::T* row, int kb, int K, int& byte) {
    constexpr int W = DT == F32 ? 2 : 1;
    u32x4 u[4 * W];
    if (kb + 32 <= K) {
        #pragma unroll
        for (int i = 0; i < 4; ++i) load8<DT>(row + kb + i * 8, u + i * W);
    } else {
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            load8_tail<DT>(row + kb + i * 8, K - kb - i * 8, u + i * W);
    }
    byte = (int)scale_byte<DT>(absmax_bits<DT>(u, 4 * W));
    const float s = scale_f32((unsigned)byte);
    i32x4 c;
    #pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (int)codes8<DT>(u + i * W, s);
    return c;
}

// FM x FN tiles of 16 x 16 a block. Its WV waves take every WVth step of 128 each
// and are joined in LDS, in their order. One row is bound by the weights' way from
// memory: 1x4096->4096 (9 MB) takes 4.0 us where the caches hold them, 6.1 where
// not (four waves: 4.9 and 8.7; 16: 4.3 and 5.6), 1x16384->4096 11 and 15 (20 and
// 25).
template <int AT, int OT, int FM, int FN, int WV>
__global__ __launch_bounds__(64 * WV)
void linear_rows_kernel(const void* __restrict__ xv,
                        const uint8_t* __restrict__ xs, long M, int K, int steps,
                        long ldx, const uint8_t* __restrict__ wc,
                        const uint8_t* __restrict__ ws, long N,
                        const void* __restrict__ bias, int bias_dt,
                        typename Elem<OT>::T* __restrict__ y, int nt) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, g = lane >> 4;
    const long m0 = (long)(blockIdx.x / nt) * (16 * FM);
    const long n0 = (long)(blockIdx.x % nt) * (16 * FN);
    const uint8_t* wp[FN];
    const uint8_t* wsp[FN];
    #pragma unroll
    for (int j = 0; j < FN; ++j) {
        const long n = min(n0 + (r16 >> 2) * (4 * FN) + j * 4 + (r16 & 3), N - 1);
        wp[j] = wc + n * 64 + g * 16;
        wsp[j] = ws + n * 16 + g * 4;
    }
    long xrow[FM];
    #pragma unroll
    for (int i = 0; i < FM; ++i) xrow[i] = min(m0 + i * 16 + r16, M - 1);

    f32x4 acc[FM][FN];
    #pragma unroll
    for (int i = 0; i < FM; ++i)
        #pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

    for (int s = wave; s < steps; s += WV) {
        i32x4 w[FN], x[FM];
        int wb[FN], xb[FM];
        #pragma unroll
        for (int j = 0; j < FN; ++j) {
            w[j] = *reinterpret_cast<const i32x4*>(wp[j] + (size_t)s * N * 64);
            wb[j] = wsp[j][(size_t)(s >> 2) * N * 16 + (s & 3)];
        }
        #pragma unroll
        for (int i = 0; i < FM; ++i) {
            if constexpr (AT == CODES) {
                x[i] = *reinterpret_cast<const i32x4*>(
                    reinterpret_cast<const uint8_t*>(xv)
                    + ((size_t)s * M + xrow[i]) * 64 + g * 16);
                xb[i] = xs[scale_at(M, xrow[i], s * 4 + g)];
            } else {
                using E = typename Elem<AT == CODES ? F32 : AT>::T;
                x[i] = round_block<AT == CODES ? F32 : AT>(
                    reinterpret_cast<const E*>(xv) + xrow[i] * ldx,
                    s * 128 + g * 32, K, xb[i]);
            }
        }
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    wide(w[j]), wide(x[i]), acc[i][j], 4, 4, 0, wb[j], 0, xb[i]);
    }

    __shared__ f32x4 part[WV - 1][FM * FN][64];
    if (wave) {
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                part[wave - 1][i * FN + j][lane] = acc[i][j];
    }
    __syncthreads();
    if (wave) return;
    #pragma unroll
    for (int p = 0; p < WV - 1; ++p)
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] += part[p][i * FN + j][lane];
    float b[4 * FN];
    load_bias<FN>(b, bias, bias_dt, n0 + g * (4 * FN), N);
    store_rows<OT, FM, FN>(acc, y, M, N, m0 + r16, n0 + g * (4 * FN), b);
}

template <int AT, int OT>
void launch_rows(const void* x, const uint8_t* xs, long M, long K, long ldx,
                 const uint8_t* wc, const uint8_t* ws, long N,
                 const void* bias, int bias_dt, void* y, int form,
                 hipStream_t stream) {
    #define MX4_L(FM, FN, WV) do { \
        const long mt = (M + 16 * FM - 1) / (16 * FM); \
        const long nt = (N + 16 * FN - 1) / (16 * FN); \
        hipLaunchKernelGGL((linear_rows_kernel<AT, OT, FM, FN, WV>), \
            dim3((unsigned)(mt * nt)), dim3(64 * WV), 0, stream, x, xs, M, (int)K, \
            (int)steps_of(K), ldx, wc, ws, N, bias, bias_dt, (typename Elem<OT>::T*)y, \
            (int)nt); } while (0)
    if (form != ROWS16 && form != HELD16) MX4_L(2, 2, 4);
    else if (M > 16 && (M + 15) / 16 * ((N + 15) / 16) > 256) MX4_L(1, 2, 4);
    else if (steps_of(K) >= 8) MX4_L(1, 1, 8);
    else MX4_L(1, 1, 4);
    #undef MX4_L
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace

// The choice; times in us, bf16, on an MI355X.
//
// The smallest blocks of which every one of 256 units has one at most: 16 x 16,
// 64x4096->1024 (256 of them) 6.7 us, 8.3 in 16 x 32 and 12.4 in 32 x 32; 16 x 32,
// 196x2048->512 (208) 5.4 against 6.7 and 7.5; 32 x 32, 784x1024->256 (200) 5.2 against
// 6.7 and 5.4.
static bool small_blocks(long M, long N) {
    return M <= 16 || (M + 15) / 16 * ((N + 31) / 32) <= 256;
}

// Rounding in the blocks saves a launch (4 us) and a pass over x, but every block
// rounds its rows again: with few multiplications M K N (16 rows count at least)
// 784x1024->256 takes 5.4 against 8.4 with the rounding before, 128x2048->2048
// (2^29) 7.6 against 8.0, 196x2048->2048 12.5 against 10.0, a longer sum
// 64x4096->2048 (2^29) 12.4 against 10.0.
//
// Many rows and few columns: x's way from memory counts, and tiles of 64 rows
// round it on the way: 62720x1024->256 35 against 42, 131072x256->64 15 against
// 24, 8192x512->256 7.7 against 10.5. There have to be blocks enough to cover a
// long sum's waits: 8192x1024->128 10.2 against 13.0 but 8192x2048->128 22 against
// 18, 32768x4096->128 56 against 77. With more columns x is rounded again:
// 16384x512->512 11.6 against 15.3, 131072x512->512 74 against 69; where the sum is
// short that does not matter, 2048x64->2048 5.6 against 8.4, 8551x12->1611 18 against
// 20 (and 39 in small blocks), until the results' way out counts, where tiles of
// more rows do better: 62720x256->1024 46 against 41, 131072x64->256 26 against 29 but
// 1003520x64->256 255 against 172.
static bool rounds_on_the_way(long M, long K, long N) {
    if (K <= 256 && M <= 16384 && (M + 31) / 32 * ((N + 31) / 32) >= 1536) return true;
    if (M < (K <= 512 ? 4096 : K <= 1024 ? 8192 : 32768)) return false;
    if (N <= 64) return true;
    if (N <= 256) return K >= 256 || M <= 131072;
    return N <= 512 && M <= 32768 && K <= 512;
}

int linear_form(long M, long K, long N) {
    if (rounds_on_the_way(M, K, N)) return ROUNDING;
    const double work = (double)(M > 16 ? M : 16) * K * N;
    if (work <= (K <= 2048 ? 0x1p29 : 0x1p28))
        return small_blocks(M, N) ? ROWS16 : ROWS32;
    return linear_q_form(M, K, N);
}

// Small blocks share a sum among their waves and read past LDS: 128x4096->4096 (2^31)
// 11.5 us against 16.7 with tiles of 128. They lose where they read too much,
// 256x4096->4096 20.8 against 16.7, or are so many that tiles fill the card (and are
// full themselves): 2048x512->1024 (2048 blocks) 7.5 against 6.0, 65536x32->128 11.3
// against 7.4; but 1024^3 (1024) 7.1 and 7.0, 64337x635->11 (2011, its tiles all but
// empty) 6.8 against 8.0. Tiles of 256 take half the bytes a result, but there have
// to be some for each of 256 units: 8192x4096->16384 (2048 tiles) 262 against 318,
// 2048x4096->4096 (128 tiles) 34 against 25; with 128 columns half of a tile is
// empty, 250880x512->128 31 against 24.
int linear_q_form(long M, long K, long N) {
    if (M <= 16) return HELD16;
    const long blocks = (M + 31) / 32 * ((N + 31) / 32);
    const bool many = blocks >= 1536 && (M + 127) / 128 * ((N + 127) / 128) * 12 <= blocks;
    if ((double)M * K * N <= 0x1p31 && !many)
        return small_blocks(M, N) ? HELD16 : HELD32;
    const long tiles = (M + 255) / 256 * ((N + 255) / 256);
    return N > 128 && tiles >= 384 ? TILES256 : TILES128;
}

size_t linear_bytes(int form, long M, long K) {
    if (form < HELD16) return 0;
    return up256(code_bytes(M, K)) + scale_bytes(M, K);
}

void linear(const void* x, int dt, long M, long K, long ldx,
            const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
            int bias_dt, void* y, int form, void* work, hipStream_t stream) {
    if (form == ROUNDING) {
        rounding(x, dt, M, K, ldx, wc, ws, N, bias, bias_dt, y, stream);
        return;
    }
    if (form >= HELD16) {
        uint8_t* xc = (uint8_t*)work;
        uint8_t* xs = xc + up256(code_bytes(M, K));
        quantize(x, dt, M, K, ldx, xc, xs, stream);
        linear_q(xc, xs, M, K, wc, ws, N, bias, bias_dt, y, dt, form, stream);
        return;
    }
    #define MX4_ARGS x, nullptr, M, K, ldx, wc, ws, N, bias, bias_dt, y, form, stream
    if (dt == F32) launch_rows<F32, F32>(MX4_ARGS);
    else if (dt == BF16) launch_rows<BF16, BF16>(MX4_ARGS);
    else launch_rows<F16, F16>(MX4_ARGS);
    #undef MX4_ARGS
}

void linear_q(const uint8_t* xc, const uint8_t* xs, long M, long K,
              const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
              int bias_dt, void* y, int dt, int form, hipStream_t stream) {
    if (form >= TILES128) {
        tiles(xc, xs, M, K, wc, ws, N, bias, bias_dt, y, dt,
              form == TILES256, stream);
        return;
    }
    #define MX4_ARGS xc, xs, M, K, 0, wc, ws, N, bias, bias_dt, y, form, stream
    if (dt == F32) launch_rows<CODES, F32>(MX4_ARGS);
    else if (dt == BF16) launch_rows<CODES, BF16>(MX4_ARGS);
    else launch_rows<CODES, F16>(MX4_ARGS);
    #undef MX4_ARGS
}

}  // namespace mx4
