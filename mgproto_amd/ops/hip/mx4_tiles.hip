// Large products of rows that are held in 4 bits: y = X W^T + bias.
//
// A block of 256 x 256 of y takes 32 KB of codes a step of 128 and 256 matrix
// instructions of 16 cycles on each of its four units, so that the bytes have
// to come from L2 at half of what a unit can take and all of it has to overlap.
// Hence
//  * a ring of S buffers in LDS, filled past the registers S - 1 steps ahead,
//    across the ends of tiles: blocks stay and walk over their tiles, so that
//    the next tile's bytes come while this one's results leave;
//  * one barrier a step, and waits that count the copies still under way
//    instead of waiting for all of them;
//  * scale words of four steps at a time: one 32-bit read a row.
// Copies from rows of 64 bytes at a distance, instead of the one piece that the
// storage gives, went at half the rate (33 against 61 bytes a cycle).

#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

template <int OT, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN)
void tiles_kernel(const uint8_t* __restrict__ xc, const uint8_t* __restrict__ xs,
                  long M, int steps, const uint8_t* __restrict__ wc,
                  const uint8_t* __restrict__ ws, long N,
                  const void* __restrict__ bias, int bias_dt,
                  typename Elem<OT>::T* __restrict__ y, int mt, int nt,
                  int group) {
    constexpr int WAVES = WM * WN, R = BM + BN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int XQ = BM / 16 / WAVES, WQ = BN / 16 / WAVES;   // copies a step
    constexpr int SQ = R / 64 / WAVES;                          // ... four steps
    static_assert(BM % (16 * WAVES) == 0 && BN % (16 * WAVES) == 0 &&
                  R % (64 * WAVES) == 0 && BM % 64 == 0, "whole copies");
    // the ring of codes, and two buffers of scales. (One array: with two the
    // compiler waits for all copies before it reads.)
    __shared__ __attribute__((aligned(16))) uint8_t lds[S * R * 64 + 2 * R * 16];
    uint8_t* const scales = lds + S * R * 64;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int wm = (wave / WN) * (FM * 16), wn = (wave % WN) * (FN * 16);

    // Blocks go round the 8 dies. Each die has a run of tiles, so that its L2
    // sees the same rows again, `group` rows of tiles at a time.
    const int total = mt * nt, xcd = blockIdx.x & 7;
    const int q8 = total >> 3, r8 = total & 7, stride = gridDim.x >> 3;
    const int lo = xcd * q8 + min(xcd, r8), hi = lo + q8 + (xcd < r8);
    auto place = [&](int t, long& m0, long& n0) {
        const int width = group * nt, first = t / width * group;
        const int rows = min(mt - first, group), in = t % width;
        m0 = (long)(first + in % rows) * BM;
        n0 = (long)(in / rows) * BN;
    };

    // what is sent for next: step lk of tile lt
    int lt = lo + (blockIdx.x >> 3), lk = 0;
    const uint8_t *lx = xc, *lw = wc, *lxs = xs, *lws = ws;
    int xo[XQ], wo[WQ], so[SQ];
    auto aim = [&]() {
        long m0, n0;
        place(lt, m0, n0);
        const int lastx = (int)min((long)BM, M - m0) - 1;
        const int lastw = (int)min((long)BN, N - n0) - 1;
        lx = xc + m0 * 64, lw = wc + n0 * 64, lxs = xs + m0 * 16, lws = ws + n0 * 16;
        #pragma unroll
        for (int q = 0; q < XQ; ++q) {
            const int r = (q * WAVES + wave) * 16 + (lane >> 2);
            xo[q] = min(r, lastx) * 64 + ((lane & 3) ^ x_key(r)) * 16;
        }
        #pragma unroll
        for (int q = 0; q < WQ; ++q) {
            const int r = (q * WAVES + wave) * 16 + (lane >> 2);
            wo[q] = min(r, lastw) * 64 + ((lane & 3) ^ w_key<FN>(r)) * 16;
        }
        #pragma unroll
        for (int q = 0; q < SQ; ++q) {
            const int r = (q * WAVES + wave) * 64 + lane;
            so[q] = (r < BM ? min(r, lastx) : min(r - BM, lastw)) * 16;
        }
    };
    int lc = 0;                                   // buffer of the next scales
    auto send = [&](int buf) {
        if ((lk & 3) == 0) {
            #pragma unroll
            for (int q = 0; q < SQ; ++q) {
                const int call = q * WAVES + wave;
                copy16_to_lds((call < BM / 64 ? lxs : lws) + (unsigned)so[q],
                              scales + lc * (R * 16) + call * 1024);
            }
            lxs += M * 16, lws += N * 16, lc ^= 1;
        }
        #pragma unroll
        for (int q = 0; q < XQ; ++q)
            copy16_to_lds(lx + (unsigned)xo[q],
                          lds + buf * (R * 64) + (q * WAVES + wave) * 1024);
        #pragma unroll
        for (int q = 0; q < WQ; ++q)
            copy16_to_lds(lw + (unsigned)wo[q],
                          lds + buf * (R * 64) + BM * 64 + (q * WAVES + wave) * 1024);
        lx += M * 64, lw += N * 64;
        if (++lk == steps) {
            lk = 0, lt += stride;
            if (lt < hi) aim();
        }
    };
    if (lt < hi && steps) {
        aim();
        #pragma unroll
        for (int b = 0; b < S - 1; ++b)
            if (lt < hi) send(b);
    }

    // Where this lane reads: rows 16 apart (x) and 4 apart (W) have the same
    // key, so that one place and constants give all of them.
    const int xr = wm + r16, wr = wn + (r16 >> 2) * (4 * FN) + (r16 & 3);
    const int xp = xr * 64 + ((g ^ x_key(xr)) << 4);
    const int wp = (BM + wr) * 64 + ((g ^ w_key<FN>(wr)) << 4);
    const int xsp = xr * 16 + g * 4, wsp = (BM + wr) * 16 + g * 4;
    int buf = 0, sbuf = 0;
    for (int t = lo + (blockIdx.x >> 3); t < hi; t += stride) {
        f32x4 acc[FM][FN];
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            #pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};
        int xb[FM], wb[FN];

        for (int k = 0; k < steps; ++k) {
            // This step's bytes have arrived: what was sent for the S - 2
            // steps behind it may still be under way (and what left since,
            // results of the last tile, came after it). Then every wave is done
            // with the buffer of the step before, which is filled again.
            const bool more = lt < hi;
            if (more)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)"
                             :: "n"((S - 2) * (XQ + WQ)) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (more) send(buf == 0 ? S - 1 : buf - 1);
            const uint8_t* c = lds + buf * (R * 64);
            if ((k & 3) == 0) {
                #pragma unroll
                for (int j = 0; j < FN; ++j)
                    wb[j] = *reinterpret_cast<const int*>(scales + sbuf * (R * 16) + wsp + j * 64);
                #pragma unroll
                for (int i = 0; i < FM; ++i)
                    xb[i] = *reinterpret_cast<const int*>(scales + sbuf * (R * 16) + xsp + i * 256);
                sbuf ^= 1;
            } else {                              // the next byte of each
                #pragma unroll
                for (int j = 0; j < FN; ++j) wb[j] = (unsigned)wb[j] >> 8;
                #pragma unroll
                for (int i = 0; i < FM; ++i) xb[i] = (unsigned)xb[i] >> 8;
            }
            i32x4 w[FN];
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                w[j] = *reinterpret_cast<const i32x4*>(c + wp + j * 256);
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                const i32x4 x = *reinterpret_cast<const i32x4*>(c + xp + i * 1024);
                #pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wide(w[j]), wide(x), acc[i][j], 4, 4, 0, wb[j], 0, xb[i]);
            }
            // reads run two rows ahead of the matrix instructions
            __builtin_amdgcn_sched_group_barrier(0x100, FN + 2, 0);
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x8, FN, 0);
                if (i + 2 < FM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            buf = buf == S - 1 ? 0 : buf + 1;
        }

        long m0, n0;
        place(t, m0, n0);
        const long n = n0 + wn + g * (4 * FN);
        float b[4 * FN];
        load_bias<FN>(b, bias, bias_dt, n, N);
        store_rows<OT, FM, FN>(acc, y, M, N, m0 + wm + r16, n, b);
    }
}

template <int OT, int BM, int BN, int WM, int WN, int S>
void launch_tiles(const uint8_t* xc, const uint8_t* xs, long M, long K,
                  const uint8_t* wc, const uint8_t* ws, long N,
                  const void* bias, int bias_dt, void* y, int blocks,
                  int group, hipStream_t stream) {
    const int mt = (int)((M + BM - 1) / BM), nt = (int)((N + BN - 1) / BN);
    const int grid = std::min((mt * nt + 7) / 8 * 8, blocks);
    hipLaunchKernelGGL((tiles_kernel<OT, BM, BN, WM, WN, S>), dim3(grid),
                       dim3(64 * WM * WN), 0, stream, xc, xs, M,
                       (int)steps_of(K), wc, ws, N, bias, bias_dt,
                       (typename Elem<OT>::T*)y, mt, nt, group);
}

}  // namespace

void tiles(const uint8_t* xc, const uint8_t* xs, long M, long K,
           const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
           int bias_dt, void* y, int dt, bool large, hipStream_t stream) {
    // 256 units: one block of 147 KB of LDS each, or two of 73 KB
    #define MX4_L(OT) \
        launch_tiles<OT, 256, 256, 2, 4, 4>(xc, xs, M, K, wc, ws, N, bias, \
                                            bias_dt, y, 256, 2, stream)
    #define MX4_S(OT) \
        launch_tiles<OT, 128, 128, 2, 2, 4>(xc, xs, M, K, wc, ws, N, bias, \
                                            bias_dt, y, 512, 4, stream)
    if (large) {
        if (dt == F32) MX4_L(F32);
        else if (dt == BF16) MX4_L(BF16);
        else MX4_L(F16);
    } else {
        if (dt == F32) MX4_S(F32);
        else if (dt == BF16) MX4_S(BF16);
        else MX4_S(F16);
    }
    #undef MX4_L
    #undef MX4_S
}

}  // namespace mx4
