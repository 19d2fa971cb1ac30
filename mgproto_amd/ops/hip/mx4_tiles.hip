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
// 8192x4096->16384 takes 262 to 290 us (4.2 to 3.8 PFLOP/s; the clock follows the
// values), 50 of them for the results, whose stores nothing overlaps.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

template <int OT, int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN, 2)
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
                  R % (64 * WAVES) == 0 && BM % 64 == 0 &&
                  FM % (XQ + WQ) == 0 && S >= 3, "whole copies");
    // The ring of codes, and as many buffers of scales: where a tile is one
    // step long, every step brings its own.
    __shared__ __attribute__((aligned(16))) uint8_t lds[S * (R * 64 + R * 16)];
    uint8_t* const scales = lds + S * R * 64;
    const unsigned to = lds_address(lds);
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
    bool more = true;                             // anything left to send
    auto send_scales = [&]() {
        if (lk & 3 || !more) return;
        #pragma unroll
        for (int q = 0; q < SQ; ++q) {
            const int call = q * WAVES + wave;
            copy16_to_lds(call < BM / 64 ? lxs : lws, (unsigned)so[q],
                          to + S * R * 64 + lc * (R * 16) + call * 1024);
        }
        lxs += M * 16, lws += N * 16, lc = lc == S - 1 ? 0 : lc + 1;
    };
    auto send_codes = [&](int buf, int q) {       // one copy of XQ + WQ
        if (q < XQ)
            copy16_to_lds(lx, (unsigned)xo[q],
                          to + buf * (R * 64) + (q * WAVES + wave) * 1024);
        else
            copy16_to_lds(lw, (unsigned)wo[q - XQ],
                          to + buf * (R * 64) + BM * 64
                              + ((q - XQ) * WAVES + wave) * 1024);
    };
    // Behind the last step the same bytes are sent again and again, so that
    // the count of copies stays what the waits take it for.
    auto sent = [&]() {
        if (!more) return;
        lx += M * 64, lw += N * 64;
        if (++lk == steps) {
            lk = 0;
            more = lt + stride < hi;
            if (more) lt += stride;
            aim();
        }
    };
    if (lt >= hi || !steps) {
        if (lt >= hi) return;
        more = false;
    } else {
        aim();
        #pragma unroll
        for (int b = 0; b < S - 1; ++b) {
            if (b) sent();
            send_scales();
            #pragma unroll
            for (int q = 0; q < XQ + WQ; ++q) send_codes(b, q);
        }
    }

    // Where this lane reads: rows 16 apart (x) and 4 apart (W) have the same
    // key, so that one place and constants give all of them.
    const int xr = wm + r16, wr = wn + (r16 >> 2) * (4 * FN) + (r16 & 3);
    const int xp = xr * 64 + ((g ^ x_key(xr)) << 4);
    const int wp = (BM + wr) * 64 + ((g ^ w_key<FN>(wr)) << 4);
    const int xsp = xr * 16 + g * 4, wsp = (BM + wr) * 16 + g * 4;
    int buf = 0, sbuf = 0;
    int xb[FM], wb[FN];
    i32x4 w[FN], x[FM];
    // the first reads of a step, made while the step before still computes
    auto begin = [&](int buf) {
        const uint8_t* c = lds + buf * (R * 64);
        #pragma unroll
        for (int j = 0; j < FN; ++j)
            w[j] = *reinterpret_cast<const i32x4*>(c + wp + j * 256);
        x[0] = *reinterpret_cast<const i32x4*>(c + xp);
        x[1] = *reinterpret_cast<const i32x4*>(c + xp + 1024);
    };
    wait_copies<0>();
    __syncthreads();
    begin(0);
    for (int t = lo + (blockIdx.x >> 3); t < hi; t += stride) {
        f32x4 acc[FM][FN];
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            #pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

        for (int k = 0; k < steps; ++k) {
            // The bytes of the step behind this one have arrived: only what was
            // sent for the S - 3 steps after it may still be under way (and
            // what left since, results of the last tile, came later). Then
            // every wave is done with the buffer of the step before this one,
            // which is filled again.
            wait_copies<(S - 3) * (XQ + WQ)>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int free = buf == 0 ? S - 1 : buf - 1;
            const uint8_t* c = lds + buf * (R * 64);
            buf = buf == S - 1 ? 0 : buf + 1;
            sent();
            send_scales();
            if ((k & 3) == 0) {
                const uint8_t* s = scales + sbuf * (R * 16);
                #pragma unroll
                for (int j = 0; j < FN; ++j)
                    wb[j] = *reinterpret_cast<const int*>(s + wsp + j * 64);
                #pragma unroll
                for (int i = 0; i < FM; ++i)
                    xb[i] = *reinterpret_cast<const int*>(s + xsp + i * 256);
                sbuf = sbuf == S - 1 ? 0 : sbuf + 1;
            } else {                              // the next byte of each
                #pragma unroll
                for (int j = 0; j < FN; ++j) wb[j] = (unsigned)wb[j] >> 8;
                #pragma unroll
                for (int i = 0; i < FM; ++i) xb[i] = (unsigned)xb[i] >> 8;
            }
            // reads two rows ahead of the matrix instructions, and the copies
            // spread among these, so that neither holds them up
            constexpr int EACH = FM / (XQ + WQ);
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (i + 2 < FM)
                    x[i + 2] = *reinterpret_cast<const i32x4*>(
                        c + xp + (i + 2) * 1024);
                if (i % EACH == 0) send_codes(free, i / EACH);
                #pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wide(w[j]), wide(x[i]), acc[i][j], 4, 4, 0, wb[j], 0, xb[i]);
            }
            begin(buf);
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (i + 2 < FM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (i == FM - 1) __builtin_amdgcn_sched_group_barrier(0x100, FN + 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, FN, 0);
            }
        }

        long m0, n0;
        place(t, m0, n0);
        const long n = n0 + wn + g * (4 * FN);
        float b[4 * FN];
        load_bias<FN>(b, bias, bias_dt, n, N);
        store_rows<OT, FM, FN>(acc, y, M, N, m0 + wm + r16, n, b);
    }
    wait_copies<0>();      // no copy is under way when LDS is given up
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
    // 256 units: one block with all 160 KB of LDS each, or two
    #define MX4_L(OT) \
        launch_tiles<OT, 256, 256, 2, 4, 4>(xc, xs, M, K, wc, ws, N, bias, \
                                            bias_dt, y, 256, 4, stream)
    #define MX4_S(OT) \
        launch_tiles<OT, 128, 128, 2, 2, 4>(xc, xs, M, K, wc, ws, N, bias, \
                                            bias_dt, y, 512, 8, stream)
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
