// Large products of 4-bit rows, tiled through LDS: y = Q(x) W^T + bias.
//
// A block sums BM x BN of y over steps of 256 elements (128 bytes of codes and
// 8 scale bytes a row). Two buffers: while the matrix cores work on one, the
// next step's codes go from memory into the other without passing registers;
// where x is still in floats, it is loaded into registers, rounded there (four
// lanes share a block, two lane exchanges for its maximum) and written as
// codes. One barrier a step.
//
// A lane's operand of v_mfma_scale_f32_16x16x128 is one block of 32, so a read
// is 16 bytes of 16 rows at once: piece c of row r lies at c ^ key(r), which
// spreads any 8 (and any 16) of these rows over all banks. In a step the lane
// group g takes pieces 2g and 2g+1, whose two scale bytes lie side by side: one
// 16-bit read gives both, and the instruction picks its byte.

#include <hip/hip_runtime.h>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

constexpr int CODES = -1;

template <int BM, int BN> struct Tile {
    uint8_t xc[BM * 128], wc[BN * 128];
    uint8_t xs[BM * 8], ws[BN * 8];
};

#define MX4_GLOBAL(p) (const __attribute__((address_space(1))) void*)(uintptr_t)(p)
#define MX4_LDS(p) (__attribute__((address_space(3))) void*)(uint32_t)(uintptr_t)(p)
// lane i's bytes go to l + i * 16 (or 4), l the same in the wave
static __device__ __forceinline__ void copy16_to_lds(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds(MX4_GLOBAL(g), MX4_LDS(l), 16, 0, 0);
}
static __device__ __forceinline__ void copy4_to_lds(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds(MX4_GLOBAL(g), MX4_LDS(l), 4, 0, 0);
}

// rows of x are read 16 consecutive ones at a time
static __device__ __forceinline__ int x_key(int r) { return (r ^ (r >> 3 & 1)) & 7; }
// rows of W in four runs of four, 4*FN apart
template <int FN> static __device__ __forceinline__ int w_key(int r) {
    const int a = r / (4 * FN);
    return ((r & 3) | (a & 1) << 2) ^ (a >> 1 & 1);
}

template <int AT, bool VEC, int OT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN)
void linear_tiled_kernel(const void* __restrict__ xv,
                         const uint8_t* __restrict__ xs, long M, int K, int Kp,
                         long ldx, const uint8_t* __restrict__ wc,
                         const uint8_t* __restrict__ ws, long N,
                         const void* __restrict__ bias, int bias_dt,
                         typename Elem<OT>::T* __restrict__ y, int mt, int nt,
                         int group) {
    using T = typename Elem<OT>::T;
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    __shared__ __attribute__((aligned(16))) Tile<BM, BN> lds[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r16 = lane & 15, g = lane >> 4;
    const int wm = (wave / WN) * (FM * 16), wn = (wave % WN) * (FN * 16);

    // Blocks go round the 8 dies; each takes a run of tiles, so that its L2
    // sees the same rows again, `group` rows of tiles at a time.
    long m0, n0;
    {
        const int total = mt * nt, xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
        const int q = total >> 3, r = total & 7;
        const int t = xcd * q + min(xcd, r) + i;
        const int width = group * nt, first = t / width * group;
        const int rows = min(mt - first, group), in = t % width;
        m0 = (long)(first + in % rows) * BM;
        n0 = (long)(in / rows) * BN;
    }
    const int cb = Kp >> 1, sb = Kp >> 5;
    const int steps = (Kp + 255) >> 8;
    const bool half = Kp & 128;              // the last step is 128 long

    // Codes of `rows` rows from row0 on, 8 rows of 128 bytes a wave's copy,
    // and 32 rows of two scale words. Offsets from the tile's first row stay
    // below 2^31 (rows are at most 2^22 long).
    auto stage_codes = [&](const uint8_t* c, const uint8_t* s, long row0,
                           long rows, uint8_t* lc, uint8_t* lsc, auto count,
                           auto key, int kt) {
        constexpr int R = decltype(count)::value;
        const int mask = half && kt == steps - 1 ? 3 : 7;
        const int last = (int)min((long)R, rows - row0) - 1;
        const uint8_t* c0 = c + row0 * cb + kt * 128;
        const uint8_t* s0 = s + row0 * sb + kt * 8;
        #pragma unroll
        for (int q = 0; q < R / 8 / WAVES; ++q) {
            const int call = q * WAVES + wave;
            const int r = call * 8 + (lane >> 3);
            const int p = ((lane & 7) ^ key(r)) & mask;
            copy16_to_lds(c0 + (unsigned)(min(r, last) * cb + p * 16),
                          lc + call * 1024);
        }
        #pragma unroll
        for (int q = 0; q < (R / 32 + WAVES - 1) / WAVES; ++q) {
            const int call = q * WAVES + wave;
            if (R / 32 % WAVES && call >= R / 32) break;
            const int r = call * 32 + (lane >> 1);
            copy4_to_lds(s0 + (unsigned)(min(r, last) * sb
                                         + (mask == 3 ? 0 : (lane & 1) * 4)),
                         lsc + call * 256);
        }
    };

    // x in floats: 8 elements a unit, 32 units a row
    constexpr int ET = AT == CODES ? F32 : AT;
    constexpr int EW = ET == F32 ? 2 : 1;
    constexpr int UNITS = AT == CODES ? 1 : BM * 32 / THREADS;
    u32x4 raw[UNITS][EW];
    auto load_x = [&](int kt) {
        using E = typename Elem<ET>::T;
        const E* x0 = reinterpret_cast<const E*>(xv) + m0 * ldx;
        const int lastx = (int)min((long)BM, M - m0) - 1;
        #pragma unroll
        for (int q = 0; q < UNITS; ++q) {
            const int u = q * THREADS + tid, r = u >> 5;
            const int k = kt * 256 + (u & 31) * 8;
            const E* p = x0 + min(r, lastx) * ldx + k;
            if (VEC && k + 8 <= K) {
                #pragma unroll
                for (int i = 0; i < EW; ++i)
                    raw[q][i] = reinterpret_cast<const u32x4*>(p)[i];
            } else {
                load8_tail<ET>(p, K - k, raw[q]);
            }
        }
    };
    auto store_x = [&](Tile<BM, BN>& t) {
        #pragma unroll
        for (int q = 0; q < UNITS; ++q) {
            const int u = q * THREADS + tid, r = u >> 5, c8 = u & 31;
            unsigned m = absmax_bits<ET>(raw[q], EW);
            m = quad_max(m);
            const unsigned byte = scale_byte<ET>(m);
            const unsigned c = codes8<ET>(raw[q], scale_f32(byte));
            *reinterpret_cast<unsigned*>(
                t.xc + r * 128 + (((c8 >> 2) ^ x_key(r)) << 4) + (c8 & 3) * 4) = c;
            if ((c8 & 3) == 0) t.xs[r * 8 + (c8 >> 2)] = (uint8_t)byte;
        }
    };
    auto stage = [&](int kt, int buf) {
        Tile<BM, BN>& t = lds[buf];
        stage_codes(wc, ws, n0, N, t.wc, t.ws, std::integral_constant<int, BN>(),
                    [](int r) { return w_key<FN>(r); }, kt);
        if constexpr (AT == CODES)
            stage_codes((const uint8_t*)xv, xs, m0, M, t.xc, t.xs,
                        std::integral_constant<int, BM>(), x_key, kt);
        else
            load_x(kt);
    };

    f32x4 acc[FM][FN];
    #pragma unroll
    for (int i = 0; i < FM; ++i)
        #pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

    // Where this lane reads: rows 16 apart (x) and 4 apart (W) have the same
    // key, so that one place and constants give all of them.
    const int xr = wm + r16, wr = wn + (r16 >> 2) * (4 * FN) + (r16 & 3);
    // pieces and scale bytes: 2g + s of a whole step, g of a half one
    auto compute = [&](const Tile<BM, BN>& t, auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        int wb[FN], xb[FM];
        #pragma unroll
        for (int j = 0; j < FN; ++j)
            wb[j] = WHOLE ? *reinterpret_cast<const unsigned short*>(
                                t.ws + wr * 8 + 2 * g + j * 32)
                          : t.ws[wr * 8 + g + j * 32];
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            xb[i] = WHOLE ? *reinterpret_cast<const unsigned short*>(
                                t.xs + xr * 8 + 2 * g + i * 128)
                          : t.xs[xr * 8 + g + i * 128];
        #pragma unroll
        for (int s = 0; s < (WHOLE ? 2 : 1); ++s) {
            const int p = WHOLE ? 2 * g + s : g;
            const uint8_t* wp = t.wc + wr * 128 + ((p ^ w_key<FN>(wr)) << 4);
            const uint8_t* xp = t.xc + xr * 128 + ((p ^ x_key(xr)) << 4);
            i32x4 w[FN];
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                w[j] = *reinterpret_cast<const i32x4*>(wp + j * 512);
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                const i32x4 x = *reinterpret_cast<const i32x4*>(xp + i * 2048);
                #pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = s == 0
                        ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                              wide(w[j]), wide(x), acc[i][j], 4, 4, 0, wb[j], 0, xb[i])
                        : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                              wide(w[j]), wide(x), acc[i][j], 4, 4, 1, wb[j], 1, xb[i]);
            }
        }
    };

    if (steps) {
        stage(0, 0);
        if constexpr (AT != CODES) store_x(lds[0]);
    }
    // Waits until a step's bytes have arrived and no wave reads the other
    // buffer any more, and sends for the next step.
    auto turn = [&](int kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (kt + 1 < steps) stage(kt + 1, (kt + 1) & 1);
    };
    const int whole = Kp >> 8;
    for (int kt = 0; kt < whole; ++kt) {
        turn(kt);
        compute(lds[kt & 1], std::true_type());
        if constexpr (AT != CODES)
            if (kt + 1 < steps) store_x(lds[(kt + 1) & 1]);
    }
    if (half) {
        turn(whole);
        compute(lds[whole & 1], std::false_type());
    }

    // a lane holds 4*FN consecutive columns of each of its FM rows
    store_rows<OT, FM, FN>(acc, y, M, N, m0 + wm + r16, n0 + wn + g * (4 * FN),
                           bias, bias_dt);
}

template <int AT, bool VEC, int OT, int BM, int BN, int WM, int WN>
void launch_tiled(const void* x, const uint8_t* xs, long M, long K, long ldx,
                  const uint8_t* wc, const uint8_t* ws, long N,
                  const void* bias, int bias_dt, void* y, int group,
                  hipStream_t stream) {
    const int Kp = (int)((K + 127) / 128 * 128);
    const int mt = (int)((M + BM - 1) / BM), nt = (int)((N + BN - 1) / BN);
    hipLaunchKernelGGL((linear_tiled_kernel<AT, VEC, OT, BM, BN, WM, WN>),
                       dim3((unsigned)(mt * nt)), dim3(64 * WM * WN), 0, stream,
                       x, xs, M, (int)K, Kp, ldx, wc, ws, N, bias, bias_dt,
                       (typename Elem<OT>::T*)y, mt, nt, group);
}

}  // namespace

void tiled_q(const uint8_t* xc, const uint8_t* xs, long M, long K,
             const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
             int bias_dt, void* y, int dt, bool large, hipStream_t stream) {
    #define MX4_T(OT, BM, BN) \
        launch_tiled<CODES, true, OT, BM, BN, 2, BN / 64>( \
            xc, xs, M, K, 0, wc, ws, N, bias, bias_dt, y, 8, stream)
    if (large) {
        if (dt == F32) MX4_T(F32, 256, 256);
        else if (dt == BF16) MX4_T(BF16, 256, 256);
        else MX4_T(F16, 256, 256);
    } else {
        if (dt == F32) MX4_T(F32, 128, 128);
        else if (dt == BF16) MX4_T(BF16, 128, 128);
        else MX4_T(F16, 128, 128);
    }
    #undef MX4_T
}

void tiled(const void* x, int dt, bool vec, long M, long K, long ldx,
           const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
           int bias_dt, void* y, hipStream_t stream) {
    #define MX4_T(DT, V, BM, BN, WM, WN) \
        launch_tiled<DT, V, DT, BM, BN, WM, WN>( \
            x, nullptr, M, K, ldx, wc, ws, N, bias, bias_dt, y, 1, stream)
    #define MX4_V(DT, BM, BN, WM, WN) do { \
        if (vec) MX4_T(DT, true, BM, BN, WM, WN); \
        else MX4_T(DT, false, BM, BN, WM, WN); } while (0)
    #define MX4_D(BM, BN, WM, WN) do { \
        if (dt == F32) MX4_V(F32, BM, BN, WM, WN); \
        else if (dt == BF16) MX4_V(BF16, BM, BN, WM, WN); \
        else MX4_V(F16, BM, BN, WM, WN); } while (0)
    if (N > 128) MX4_D(128, 256, 2, 4);
    else if (N > 64) MX4_D(128, 128, 4, 2);
    else MX4_D(128, 64, 8, 1);
    #undef MX4_D
    #undef MX4_V
    #undef MX4_T
}

}  // namespace mx4
