// Rows to MX4 blocks and back. See mx4_common.h for the format.
//
// Bound by memory: 2 (or 4) bytes in and 0.53 out an element, the reverse for
// reading back. Four lanes share a block, 8 elements each, and its maximum goes
// over them by two lane exchanges. A wave takes 512 elements of a row (or 128
// of four rows, where rows are that short), so that it reads in pieces of 1 KB
// or more, and four such pieces at once to have enough loads under way. Values
// read back go out past the caches (250880x512 62 -> 47 us), unless pieces of two
// rows share 16 bytes (62720x1023 26 -> 32).
// 62720x1024 bf16: rounded in 24 us, read back in 24 (6.7 TB/s each).

#include <hip/hip_runtime.h>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

constexpr int ROWS = 4;       // pieces a wave has under way

struct Rows {                 // of one matrix, and where its blocks go
    const void* x;
    long R, ldx;
    uint8_t *codes, *scales;
    int dt;
};

// LPR lanes hold a row's piece: 64 of them 512 elements, 16 of them 128
template <int DT, int LPR>
static __device__ __forceinline__ void quantize_rows(const Rows& a, int K,
                                                     int steps, int chunks,
                                                     long block) {
    constexpr int W = DT == F32 ? 2 : 1;
    constexpr int RPW = 64 / LPR;                // rows side by side
    const typename Elem<DT>::T* x = (const typename Elem<DT>::T*)a.x;
    const long R = a.R;
    const int lane = threadIdx.x & 63, sub = lane % LPR;
    const long wave = block * 4 + (threadIdx.x >> 6);
    const int chunk = (int)(wave % chunks);
    const long row0 = wave / chunks * (RPW * ROWS) + lane / LPR;
    const int k = chunk * 512 + sub * 8, s = k >> 7;
    u32x4 u[ROWS][W];
    #pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long row = row0 + i * RPW;
        const typename Elem<DT>::T* p = x + min(row, R - 1) * a.ldx + k;
        if (k + 8 <= K) load8<DT>(p, u[i]);
        else load8_tail<DT>(p, K - k, u[i]);
    }
    #pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long row = row0 + i * RPW;
        const unsigned byte = scale_byte<DT>(quad_max(absmax_bits<DT>(u[i], W)));
        const unsigned c = codes8<DT>(u[i], scale_f32(byte));
        // block g of four steps lies in lanes 4g, 4g + 16, ...; behind the
        // row the elements were zeros and so are the bytes
        unsigned four = byte;
        if constexpr (LPR == 64) {
            four |= (unsigned)__shfl((int)byte, (lane & 15) + 16) << 8;
            four |= (unsigned)__shfl((int)byte, (lane & 15) + 32) << 16;
            four |= (unsigned)__shfl((int)byte, (lane & 15) + 48) << 24;
        }
        if (row >= R) continue;
        if (s < steps)
            reinterpret_cast<unsigned*>(a.codes)[
                ((size_t)s * R + row) * 16 + (sub & 15)] = byte == 255u ? 0u : c;
        if (sub < 16 && (sub & 3) == 0)
            reinterpret_cast<unsigned*>(a.scales)[
                ((size_t)chunk * R + row) * 4 + (sub >> 2)] = four;
    }
}

// The number of this block; a grid too long for one axis has several rows of
// blocks, the last ones of which find no rows left.
static __device__ __forceinline__ long block_number() {
    return (long)blockIdx.y * gridDim.x + blockIdx.x;
}

template <int DT, int LPR>
__global__ __launch_bounds__(256)
void quantize_kernel(const Rows a, int K, int steps, int chunks) {
    quantize_rows<DT, LPR>(a, K, steps, chunks, block_number());
}

// Two matrices of the same row length, the first in the first blocks: one
// launch less for a training step, which rounds the weight and the rows.
template <int LPR>
__global__ __launch_bounds__(256)
void quantize_two_kernel(const Rows a, const Rows b, long first, int K,
                         int steps, int chunks) {
    const long number = block_number();
    const bool is_a = number < first;
    const Rows& r = is_a ? a : b;
    const long block = is_a ? number : number - first;
    if (r.dt == F32) quantize_rows<F32, LPR>(r, K, steps, chunks, block);
    else if (r.dt == BF16)
        quantize_rows<BF16, LPR>(r, K, steps, chunks, block);
    else quantize_rows<F16, LPR>(r, K, steps, chunks, block);
}

template <int DT, int LPR>
__global__ __launch_bounds__(256)
void dequantize_kernel(const uint8_t* __restrict__ codes,
                       const uint8_t* __restrict__ scales, long R, int K,
                       typename Elem<DT>::T* __restrict__ out, int chunks) {
    using T = typename Elem<DT>::T;
    constexpr int RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, sub = lane % LPR;
    const long wave = block_number() * 4 + (threadIdx.x >> 6);
    const int chunk = (int)(wave % chunks);
    const long row0 = wave / chunks * (RPW * ROWS) + lane / LPR;
    const int k = chunk * 512 + sub * 8;
    const bool whole = K % 8 == 0;
    if (k >= K) return;
    unsigned c[ROWS], byte[ROWS];
    #pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long row = min(row0 + i * RPW, R - 1);
        c[i] = reinterpret_cast<const unsigned*>(codes)[
            ((size_t)(k >> 7) * R + row) * 16 + (sub & 15)];
        byte[i] = scales[scale_at(R, row, k >> 5)];
    }
    #pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const long row = row0 + i * RPW;
        if (row >= R) continue;
        Piece<T, 8> o;
        float f[8];
        values8(c[i], byte[i], f);
        #pragma unroll
        for (int e = 0; e < 8; ++e) o.v[e] = from_f32<DT>(f[e]);
        if (whole) store_piece<true>(out + row * K + k, o, K - k);
        else store_piece(out + row * K + k, o, K - k);
    }
}

// blocks of four waves; short rows lie four side by side
long blocks_for(long R, long K, bool shortrow) {
    const long waves = shortrow ? (R + 4 * ROWS - 1) / (4 * ROWS)
                                : (R + ROWS - 1) / ROWS * chunks_of(K);
    return (waves + 3) / 4;
}

// An axis of a launch has fewer than 2^32 threads, and a block takes 16 rows of 512
// elements: 2^28 rows of 129 fill more than one.
dim3 grid_of(long blocks) {
    constexpr long MOST = 1L << 23;
    if (blocks <= MOST) return dim3((unsigned)blocks);
    return dim3((unsigned)MOST, (unsigned)((blocks + MOST - 1) / MOST));
}

}  // namespace

void quantize(const void* x, int dt, long rows, long K, long ldx,
              uint8_t* codes, uint8_t* scales, hipStream_t stream) {
    if (rows == 0 || K == 0) return;
    const bool shortrow = K <= 128;
    const Rows a{x, rows, ldx, codes, scales, dt};
    const dim3 grid = grid_of(blocks_for(rows, K, shortrow));
    #define MX4_Q(DT, L) \
        hipLaunchKernelGGL((quantize_kernel<DT, L>), grid, dim3(256), 0, stream, \
                           a, (int)K, (int)steps_of(K), (int)chunks_of(K))
    #define MX4_L(DT) do { if (shortrow) MX4_Q(DT, 16); \
                           else MX4_Q(DT, 64); } while (0)
    if (dt == F32) MX4_L(F32);
    else if (dt == BF16) MX4_L(BF16);
    else MX4_L(F16);
    #undef MX4_L
    #undef MX4_Q
}

void quantize_two(const void* x, int dt, long rows, long ldx, uint8_t* codes,
                  uint8_t* scales, const void* x2, int dt2, long rows2,
                  long ldx2, uint8_t* codes2, uint8_t* scales2, long K,
                  hipStream_t stream) {
    if (K == 0 || rows == 0 || rows2 == 0) {
        quantize(x, dt, rows, K, ldx, codes, scales, stream);
        quantize(x2, dt2, rows2, K, ldx2, codes2, scales2, stream);
        return;
    }
    const bool shortrow = K <= 128;
    const Rows a{x, rows, ldx, codes, scales, dt};
    const Rows b{x2, rows2, ldx2, codes2, scales2, dt2};
    const long first = blocks_for(rows, K, shortrow);
    const dim3 grid = grid_of(first + blocks_for(rows2, K, shortrow));
    #define MX4_Q(L) \
        hipLaunchKernelGGL((quantize_two_kernel<L>), grid, dim3(256), 0, stream, \
                           a, b, first, (int)K, (int)steps_of(K), \
                           (int)chunks_of(K))
    if (shortrow) MX4_Q(16);
    else MX4_Q(64);
    #undef MX4_Q
}

void dequantize(const uint8_t* codes, const uint8_t* scales, long rows,
                long K, void* out, int dt, hipStream_t stream) {
    if (rows == 0 || K == 0) return;
    const bool shortrow = K <= 128;
    const dim3 grid = grid_of(blocks_for(rows, K, shortrow));
    #define MX4_D(DT, L) \
        hipLaunchKernelGGL((dequantize_kernel<DT, L>), grid, dim3(256), 0, \
                           stream, codes, scales, rows, (int)K, \
                           (typename Elem<DT>::T*)out, (int)chunks_of(K))
    #define MX4_L(DT) do { if (shortrow) MX4_D(DT, 16); \
                           else MX4_D(DT, 64); } while (0)
    if (dt == F32) MX4_L(F32);
    else if (dt == BF16) MX4_L(BF16);
    else MX4_L(F16);
    #undef MX4_L
    #undef MX4_D
}

}  // namespace mx4
