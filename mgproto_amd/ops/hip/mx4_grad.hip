// Straight-through gradients of the 4-bit product:
//   dx[M,K] = g[M,N] W[N,K],   dw[N,K] = g[M,N]^T X[M,K],   db[n] = sum_m g.
//
// Every MX4 value is exact in bf16, so the held operand is read as bf16 and
// both products run on v_mfma_f32_16x16x32_bf16 with fp32 sums. g is taken
// whole: a wider type is cut into bf16 parts by truncation (two for fp16's 11
// bits, three for fp32's 24), whose sum is g exactly, and the parts' products
// are added in the same sums.

#include <hip/hip_runtime.h>

#include "mx4_common.h"
#include "mx4_linear.h"

namespace mx4 {
namespace {

constexpr int BT = 128, BK = 64;      // tile of the output, step of the sum

int parts_of(int dt) { return dt == BF16 ? 1 : dt == F16 ? 2 : 3; }
long up64(long v) { return (v + 63) / 64 * 64; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// part p of v: eight bits of its significand each time
static __device__ __forceinline__ unsigned short part_of(float v, int p) {
    unsigned b = __float_as_uint(v);
    if ((b & 0x7f800000u) == 0x7f800000u) {       // infinity or NaN: whole in
        if (p) return 0;                          // the first part
        return (unsigned short)((b >> 16) | ((b & 0x7fffffu) ? 0x40u : 0u));
    }
    for (int i = 0; i < p; ++i) {
        v -= __uint_as_float(b & 0xffff0000u);    // exact
        b = __float_as_uint(v);
    }
    return (unsigned short)(b >> 16);
}

// ---------------------------------------------------------------------------
// operands laid out for the product: rows along the summed axis, zeros up to
// a multiple of 64
// ---------------------------------------------------------------------------

// g [R, C] -> out [P][R][Cp]
template <int DT>
__global__ __launch_bounds__(256)
void parts_kernel(const typename Elem<DT>::T* __restrict__ g, long R, long C,
                  long Cp, int P, unsigned short* __restrict__ out) {
    const long total = R * Cp, step = (long)gridDim.x * 256;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
        const long r = t / Cp, c = t - r * Cp;
        const float v = c < C ? (float)g[r * C + c] : 0.f;
        for (int p = 0; p < P; ++p) out[p * total + t] = part_of(v, p);
    }
}

// g [R, C] -> out [P][C][Rp]
template <int DT>
__global__ __launch_bounds__(256)
void parts_t_kernel(const typename Elem<DT>::T* __restrict__ g, long R, long C,
                    long Rp, int P, unsigned short* __restrict__ out) {
    __shared__ float tile[64][65];
    const long r0 = (long)blockIdx.x * 64, c0 = (long)blockIdx.y * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int i = ty; i < 64; i += 4) {
        const long r = r0 + i, c = c0 + tx;
        tile[i][tx] = r < R && c < C ? (float)g[r * C + c] : 0.f;
    }
    __syncthreads();
    for (int i = ty; i < 64; i += 4) {
        const long c = c0 + i;
        if (c >= C) break;
        for (int p = 0; p < P; ++p)
            out[((long)p * C + c) * Rp + r0 + tx] = part_of(tile[tx][i], p);
    }
}

// 4-bit rows [R, K] -> out [K][Rp]
__global__ __launch_bounds__(256)
void values_t_kernel(const uint8_t* __restrict__ codes,
                     const uint8_t* __restrict__ scales, long R, long K,
                     long Rp, __bf16* __restrict__ out) {
    __shared__ float tile[64][65];
    const long r0 = (long)blockIdx.x * 64, k0 = (long)blockIdx.y * 64;
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    {   // 8 codes a thread, 32 rows at a time
        const int u = threadIdx.x & 7, rr = threadIdx.x >> 3;
        const int k = (int)k0 + u * 8;
        for (int i = rr; i < 64; i += 32) {
            const long r = r0 + i;
            unsigned c = 0, byte = 0;
            if (r < R) {                       // 64 divides a step
                c = reinterpret_cast<const unsigned*>(codes)[
                    ((size_t)(k >> 7) * R + r) * 16 + (k >> 3 & 15)];
                byte = scales[scale_at(R, r, k >> 5)];
            }
            float f[8];
            values8(c, byte, f);
            #pragma unroll
            for (int e = 0; e < 8; ++e) tile[i][u * 8 + e] = f[e];
        }
    }
    __syncthreads();
    for (int i = ty; i < 64; i += 4) {
        const long k = k0 + i;
        if (k >= K) break;
        out[k * Rp + r0 + tx] = (__bf16)tile[tx][i];
    }
}

// ---------------------------------------------------------------------------
// C[M,N] = sum_p A_p[M,Kc] B[N,Kc]^T, rows of multiples of 64 elements
// ---------------------------------------------------------------------------

// Grid (row tiles, column tiles, splits). A split sums its share of the
// steps of all parts; with more than one split C is fp32 [splits][M][N].
// LDS rows are 128 bytes; 16-byte piece c of row r lies at c ^ key(r), so
// that the 16 rows which a read takes at once fall on different banks.
static __device__ __forceinline__ int a_key(int r) { return (r ^ (r >> 3 & 1)) & 7; }
static __device__ __forceinline__ int b_key(int r) {      // runs of 4, 16 apart
    return ((r & 3) | (r >> 4 & 1) << 2) ^ (r >> 5 & 1);
}

template <int OT>
__global__ __launch_bounds__(256)
void product_nt_kernel(const unsigned short* __restrict__ A, long lda,
                       long part_stride, int P,
                       const unsigned short* __restrict__ B, long ldb,
                       long M, long N, long Kc,
                       typename Elem<OT>::T* __restrict__ C) {
    using T = typename Elem<OT>::T;
    __shared__ __attribute__((aligned(16))) unsigned short lds[2][2][BT * BK];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const long m0 = (long)blockIdx.x * BT, n0 = (long)blockIdx.y * BT;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    const long per = Kc / BK, steps = per * P;
    const long s_lo = steps * blockIdx.z / gridDim.z;
    const long s_hi = steps * (blockIdx.z + 1) / gridDim.z;
    const int lasta = (int)min((long)BT, M - m0) - 1;
    const int lastb = (int)min((long)BT, N - n0) - 1;

    // offsets in a tile stay below 2^31: rows are at most 2^22 elements here,
    // 2^31 / 256 along M (checked by the caller)
    auto stage = [&](long s, int buf) {
        const long p = s / per, k0 = (s - p * per) * BK;
        const unsigned short* a = A + p * part_stride + m0 * lda + k0;
        const unsigned short* b = B + n0 * ldb + k0;
        #pragma unroll
        for (int q = 0; q < 4; ++q) {          // 1 KB: 8 rows a wave's call
            const int call = wave * 4 + q;
            const int r = call * 8 + (lane >> 3), c = lane & 7;
            copy16_to_lds(a, (unsigned)(min(r, lasta) * lda * 2) + (c ^ a_key(r)) * 16,
                          lds_address(&lds[buf][0][call * 512]));
            copy16_to_lds(b, (unsigned)(min(r, lastb) * ldb * 2) + (c ^ b_key(r)) * 16,
                          lds_address(&lds[buf][1][call * 512]));
        }
    };

    f32x4 acc[4][4];
    #pragma unroll
    for (int i = 0; i < 4; ++i)
        #pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

    if (s_lo < s_hi) stage(s_lo, 0);
    int buf = 0;
    for (long s = s_lo; s < s_hi; ++s, buf ^= 1) {
        // the pieces of this step have to be there, and every wave has to be
        // done with the other buffer before it is filled again
        wait_copies<0>();
        __syncthreads();
        if (s + 1 < s_hi) stage(s + 1, buf ^ 1);
        #pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 a[4], b[4];
            const int c = kk * 4 + g;
            #pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = wm + i * 16 + r16;
                a[i] = *reinterpret_cast<const bf16x8*>(
                    &lds[buf][0][r * BK + (c ^ a_key(r)) * 8]);
            }
            #pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = wn + (r16 >> 2) * 16 + j * 4 + (r16 & 3);
                b[j] = *reinterpret_cast<const bf16x8*>(
                    &lds[buf][1][r * BK + (c ^ b_key(r)) * 8]);
            }
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                #pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        b[j], a[i], acc[i][j], 0, 0, 0);
        }
    }

    // a lane holds 16 consecutive columns of each of its 4 rows
    T* out = C + (gridDim.z > 1 ? (long)blockIdx.z * M * N : 0);
    const bool vec = N % 4 == 0;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long m = m0 + wm + i * 16 + r16;
        if (m >= M) continue;
        #pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long n = n0 + wn + g * 16 + j * 4;
            if (n >= N) continue;
            T* q = out + m * N + n;
            union { T v[4]; u32x2 u[sizeof(T) / 2]; } o;
            #pragma unroll
            for (int r = 0; r < 4; ++r) o.v[r] = from_f32<OT>(acc[i][j][r]);
            if (vec) {
                #pragma unroll
                for (int r = 0; r < (int)sizeof(T) / 2; ++r)
                    reinterpret_cast<u32x2*>(q)[r] = o.u[r];
            } else {
                #pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < N) q[r] = o.v[r];
            }
        }
    }
}

// out[i] = sum of the splits, in their order
template <int OT>
__global__ __launch_bounds__(256)
void join_kernel(const float* __restrict__ part, int S, long n,
                 typename Elem<OT>::T* __restrict__ out) {
    const long step = (long)gridDim.x * 256;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < n; t += step) {
        float v = 0.f;
        for (int s = 0; s < S; ++s) v += part[s * n + t];
        out[t] = from_f32<OT>(v);
    }
}

unsigned grid_for(long total) {
    const long blocks = (total + 255) / 256;
    return (unsigned)(blocks < 256 * 32 ? blocks : 256 * 32);
}

// Splits of the sum: enough blocks for two on each of 256 units, each split
// at least 4 steps long.
int splits_for(long M, long N, long steps) {
    const long tiles = ((M + BT - 1) / BT) * ((N + BT - 1) / BT);
    long s = (512 + tiles - 1) / tiles;
    if (s > steps / 4) s = steps / 4;
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}

size_t split_bytes(long M, long N, long steps) {
    const int S = splits_for(M, N, steps);
    return S > 1 ? up256((size_t)S * M * N * 4) : 0;
}

void product_nt(const unsigned short* A, long lda, long part_stride, int P,
                const unsigned short* B, long ldb, long M, long N, long Kc,
                void* out, int dt, float* part, hipStream_t stream) {
    const int S = splits_for(M, N, Kc / BK * P);
    const dim3 grid((unsigned)((M + BT - 1) / BT),
                    (unsigned)((N + BT - 1) / BT), (unsigned)S);
    #define MX4_P(DT, C) \
        hipLaunchKernelGGL((product_nt_kernel<DT>), grid, dim3(256), 0, \
                           stream, A, lda, part_stride, P, B, ldb, M, N, Kc, \
                           (typename Elem<DT>::T*)(C))
    if (S == 1) {
        if (dt == F32) MX4_P(F32, out);
        else if (dt == BF16) MX4_P(BF16, out);
        else MX4_P(F16, out);
        return;
    }
    MX4_P(F32, part);
    #undef MX4_P
    const long n = M * N;
    #define MX4_J(DT) \
        hipLaunchKernelGGL((join_kernel<DT>), dim3(grid_for(n)), dim3(256), \
                           0, stream, part, S, n, (typename Elem<DT>::T*)out)
    if (dt == F32) MX4_J(F32);
    else if (dt == BF16) MX4_J(BF16);
    else MX4_J(F16);
    #undef MX4_J
}

// ---------------------------------------------------------------------------
// column sums
// ---------------------------------------------------------------------------

constexpr int SUM_ROWS = 512;

template <int DT>
__global__ __launch_bounds__(256)
void col_sum_kernel(const typename Elem<DT>::T* __restrict__ g, long M, long N,
                    float* __restrict__ part) {
    __shared__ float red[4][64];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const long n = (long)blockIdx.x * 64 + tx;
    const long lo = (long)blockIdx.y * SUM_ROWS;
    const long hi = min(lo + SUM_ROWS, M);
    float v = 0.f;
    if (n < N)
        for (long m = lo + ty; m < hi; m += 4) v += (float)g[m * N + n];
    red[ty][tx] = v;
    __syncthreads();
    if (ty == 0 && n < N)
        part[blockIdx.y * N + n] =
            (red[0][tx] + red[1][tx]) + (red[2][tx] + red[3][tx]);
}

}  // namespace

size_t col_sum_bytes(long M, long N) {
    return up256((size_t)((M + SUM_ROWS - 1) / SUM_ROWS) * N * 4);
}

void col_sum(const void* g, int g_dt, long M, long N, void* out, int out_dt,
             void* work, hipStream_t stream) {
    const int S = (int)((M + SUM_ROWS - 1) / SUM_ROWS);
    float* part = (float*)work;
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)S);
    #define MX4_S(DT) \
        hipLaunchKernelGGL((col_sum_kernel<DT>), grid, dim3(256), 0, stream, \
                           (const typename Elem<DT>::T*)g, M, N, part)
    if (g_dt == F32) MX4_S(F32);
    else if (g_dt == BF16) MX4_S(BF16);
    else MX4_S(F16);
    #undef MX4_S
    #define MX4_J(DT) \
        hipLaunchKernelGGL((join_kernel<DT>), dim3(grid_for(N)), dim3(256), \
                           0, stream, part, S, N, (typename Elem<DT>::T*)out)
    if (out_dt == F32) MX4_J(F32);
    else if (out_dt == BF16) MX4_J(BF16);
    else MX4_J(F16);
    #undef MX4_J
}

// dx = g W: W^T is written once as [K][Np] bf16; g is read in place where its
// rows allow it, and copied into padded bf16 parts elsewhere
static bool in_place(long N, int g_dt, bool g_aligned) {
    return g_dt == BF16 && g_aligned && N % 64 == 0;
}

size_t grad_input_bytes(long M, long N, long K, int g_dt, bool g_aligned) {
    const long Np = up64(N);
    const int P = parts_of(g_dt);
    size_t b = up256((size_t)K * Np * 2);
    if (!in_place(N, g_dt, g_aligned)) b += up256((size_t)P * M * Np * 2);
    return b + split_bytes(M, K, Np / BK * P);
}

void grad_input(const void* g, int g_dt, bool g_aligned, long M, long N,
                long K, const uint8_t* wc, const uint8_t* ws, void* dx,
                int dx_dt, void* work, hipStream_t stream) {
    const long Np = up64(N);
    const int P = parts_of(g_dt);
    char* at = (char*)work;
    __bf16* wt = (__bf16*)at;
    at += up256((size_t)K * Np * 2);
    hipLaunchKernelGGL(values_t_kernel,
                       dim3((unsigned)(Np / 64), (unsigned)((K + 63) / 64)),
                       dim3(256), 0, stream, wc, ws, N, K, Np, wt);
    const unsigned short* a = (const unsigned short*)g;
    if (!in_place(N, g_dt, g_aligned)) {
        unsigned short* parts = (unsigned short*)at;
        at += up256((size_t)P * M * Np * 2);
        #define MX4_G(DT) \
            hipLaunchKernelGGL((parts_kernel<DT>), dim3(grid_for(M * Np)), \
                               dim3(256), 0, stream, \
                               (const typename Elem<DT>::T*)g, M, N, Np, P, parts)
        if (g_dt == F32) MX4_G(F32);
        else if (g_dt == BF16) MX4_G(BF16);
        else MX4_G(F16);
        #undef MX4_G
        a = parts;
    }
    product_nt(a, Np, M * Np, P, (const unsigned short*)wt, Np, M, K, Np, dx,
               dx_dt, (float*)at, stream);
}

// dw = g^T X: both turned so that rows lie along M
size_t grad_weight_bytes(long M, long N, long K, int g_dt) {
    const long Mp = up64(M);
    const int P = parts_of(g_dt);
    return up256((size_t)K * Mp * 2) + up256((size_t)P * N * Mp * 2) +
           split_bytes(N, K, Mp / BK * P);
}

void grad_weight(const void* g, int g_dt, long M, long N, long K,
                 const uint8_t* xc, const uint8_t* xs, void* dw, int dw_dt,
                 void* work, hipStream_t stream) {
    const long Mp = up64(M);
    const int P = parts_of(g_dt);
    char* at = (char*)work;
    __bf16* xt = (__bf16*)at;
    at += up256((size_t)K * Mp * 2);
    unsigned short* gt = (unsigned short*)at;
    at += up256((size_t)P * N * Mp * 2);
    hipLaunchKernelGGL(values_t_kernel,
                       dim3((unsigned)(Mp / 64), (unsigned)((K + 63) / 64)),
                       dim3(256), 0, stream, xc, xs, M, K, Mp, xt);
    const dim3 grid((unsigned)(Mp / 64), (unsigned)((N + 63) / 64));
    #define MX4_G(DT) \
        hipLaunchKernelGGL((parts_t_kernel<DT>), grid, dim3(256), 0, stream, \
                           (const typename Elem<DT>::T*)g, M, N, Mp, P, gt)
    if (g_dt == F32) MX4_G(F32);
    else if (g_dt == BF16) MX4_G(BF16);
    else MX4_G(F16);
    #undef MX4_G
    product_nt(gt, Mp, N * Mp, P, (const unsigned short*)xt, Mp, N, K, Mp, dw,
               dw_dt, (float*)at, stream);
}

}  // namespace mx4
