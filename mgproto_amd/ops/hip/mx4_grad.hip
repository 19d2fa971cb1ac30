// Straight-through gradients of the 4-bit product:
//   dx[M,K] = g[M,N] W[N,K],   dw[N,K] = g[M,N]^T X[M,K],   db[n] = sum_m g.
//
// Every MX4 value is exact in bf16, so the held operand is read as bf16 and
// both products run on bf16 matrix instructions with fp32 sums
// (mx4_grad_input.hip, mx4_grad_weight.hip). g is taken whole: a wider type is
// cut into bf16 parts by truncation (two for fp16's 11 bits, three for fp32's
// 24), whose sum is g exactly, and the parts' products are added in the same
// sums. Small products, where every launch counts, take one kernel of plain
// fp32 arithmetic instead.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_grad.h"

namespace mx4 {
namespace {

int parts_of(int dt) { return dt == BF16 ? 1 : dt == F16 ? 2 : 3; }

// part p of v: eight bits of its significand each time
static __device__ __forceinline__ unsigned part_of(float v, int p) {
    unsigned b = __float_as_uint(v);
    if ((b & 0x7f800000u) == 0x7f800000u) {       // infinity or NaN: whole in
        if (p) return 0;                          // the first part
        return (b >> 16) | ((b & 0x7fffffu) ? 0x40u : 0u);
    }
    for (int i = 0; i < p; ++i) {
        v -= __uint_as_float(b & 0xffff0000u);    // exact
        b = __float_as_uint(v);
    }
    return b >> 16;
}

// what load8 gave
template <int DT>
static __device__ __forceinline__ void floats8(const u32x4* u, float* f) {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == F32) {
            f[i] = __uint_as_float(u[0][i]);
            f[4 + i] = __uint_as_float(u[1][i]);
        } else {
            const unsigned w = u[0][i];
            f[2 * i] = DT == BF16 ? __uint_as_float(w << 16)
                                  : (float)as_f16x2(w).x;
            f[2 * i + 1] = DT == BF16 ? __uint_as_float(w & 0xffff0000u)
                                      : (float)as_f16x2(w).y;
        }
    }
}

// ---------------------------------------------------------------------------
// operands laid out for the tiles
// ---------------------------------------------------------------------------

// g [M, N] -> parts of it, 8 elements a thread: STEPPED [P][Np/32][M][32], else
// [P][M][Np]; zeros behind column N
template <int DT, bool STEPPED>
__global__ __launch_bounds__(256)
void parts_kernel(const typename Elem<DT>::T* __restrict__ g, long M, int N,
                  int Np, int P, u32x4* __restrict__ out) {
    const int upr = Np / 8;
    const long total = M * upr, step = (long)gridDim.x * 256;
    for (long t = (long)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
        const long m = t / upr;
        const int u = (int)(t - m * upr), n = u * 8;
        const typename Elem<DT>::T* q = g + m * N + n;
        u32x4 raw[DT == F32 ? 2 : 1];
        if (n + 8 <= N) load8<DT>(q, raw);
        else load8_tail<DT>(q, N - n, raw);
        float v[8];
        floats8<DT>(raw, v);
        const long at = STEPPED ? ((long)(u >> 2) * M + m) * 4 + (u & 3) : t;
        for (int p = 0; p < P; ++p) {
            u32x4 o;
            #pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = part_of(v[2 * i], p) | part_of(v[2 * i + 1], p) << 16;
            out[p * total + at] = o;
        }
    }
}

// 4-bit rows [R, K] -> [ceil(R/32)][K][32] bf16, zeros behind row R
__global__ __launch_bounds__(256)
void values_t_kernel(const uint8_t* __restrict__ codes,
                     const uint8_t* __restrict__ scales, long R, long K,
                     __bf16* __restrict__ out) {
    __shared__ float tile[32][129];
    const long r0 = (long)blockIdx.x * 32, k0 = (long)blockIdx.y * 128;
    #pragma unroll
    for (int q = 0; q < 2; ++q) {       // 32 rows of 16 words
        const int w = q * 256 + threadIdx.x, i = w >> 4, u = w & 15;
        const long r = r0 + i;
        unsigned c = 0, byte = 0;
        if (r < R) {
            c = reinterpret_cast<const unsigned*>(codes)[
                ((size_t)blockIdx.y * R + r) * 16 + u];
            byte = scales[scale_at(R, r, (int)(k0 >> 5) + (u >> 2))];
        }
        float f[8];
        values8(c, byte, f);
        #pragma unroll
        for (int e = 0; e < 8; ++e) tile[i][u * 8 + e] = f[e];
    }
    __syncthreads();
    #pragma unroll
    for (int q = 0; q < 2; ++q) {       // 128 columns of 4 pieces of 8
        const int w = q * 256 + threadIdx.x, k = w >> 2, p = w & 3;
        if (k0 + k >= K) break;
        u32x4 o;
        #pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __bf16 lo = (__bf16)tile[p * 8 + 2 * i][k];
            const __bf16 hi = (__bf16)tile[p * 8 + 2 * i + 1][k];
            o[i] = __builtin_bit_cast(unsigned short, lo)
                | (unsigned)__builtin_bit_cast(unsigned short, hi) << 16;
        }
        reinterpret_cast<u32x4*>(out)[((long)blockIdx.x * K + k0 + k) * 4 + p] = o;
    }
}

// ---------------------------------------------------------------------------
// sums of partial results
// ---------------------------------------------------------------------------

// 16 results a block; 16 groups of lanes sum a sixteenth of the parts each
template <int OT>
__global__ __launch_bounds__(256)
void join_few_kernel(const float* __restrict__ part, int S, long n,
                     typename Elem<OT>::T* __restrict__ out) {
    __shared__ float red[16][17];
    const int x = threadIdx.x & 15, q = threadIdx.x >> 4;
    const long i = (long)blockIdx.x * 16 + x;
    const int lo = S * q / 16, hi = S * (q + 1) / 16;
    float v = 0.f;
    if (i < n) {
        #pragma unroll 8
        for (int s = lo; s < hi; ++s) v += part[s * n + i];
    }
    red[q][x] = v;
    __syncthreads();
    if (q || i >= n) return;
    float s = 0.f;
    #pragma unroll
    for (int k = 0; k < 16; ++k) s += red[k][x];
    out[i] = from_f32<OT>(s);
}

// 4 results a thread; a part may start anywhere (2079x243 of 3280: 5 us for 15)
template <int OT>
__global__ __launch_bounds__(256)
void join_many_kernel(const float* __restrict__ part, int S, long n,
                      typename Elem<OT>::T* __restrict__ out) {
    using T = typename Elem<OT>::T;
    struct __attribute__((packed, aligned(4))) Four { f32x4 v; };
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 v = {0, 0, 0, 0};
    if (i + 4 <= n) {
        #pragma unroll 8
        for (int s = 0; s < S; ++s)
            v += reinterpret_cast<const Four*>(part + s * n + i)->v;
    } else {
        for (int s = 0; s < S; ++s)
            #pragma unroll
            for (int r = 0; r < 3; ++r)
                if (i + r < n) v[r] += part[s * n + i + r];
    }
    Piece<T, 4> o;
    #pragma unroll
    for (int r = 0; r < 4; ++r) o.v[r] = from_f32<OT>(v[r]);
    store_piece(out + i, o, n - i);
}

// Sums over rows: W lanes side by side take 8 columns each, 256 / W rows at a
// time; part[chunk][n]
template <int DT>
__global__ __launch_bounds__(256)
void col_sum_kernel(const typename Elem<DT>::T* __restrict__ g, long M, int N,
                    int W, long rows, float* __restrict__ part) {
    constexpr int E = DT == F32 ? 2 : 1;
    __shared__ float red[256][9];
    const int x = threadIdx.x & (W - 1), y = threadIdx.x / W, Y = 256 / W;
    const long n = ((long)blockIdx.x * W + x) * 8;
    const long lo = blockIdx.y * rows, hi = min(lo + rows, M);
    float v[8] = {};
    if (n < N) {
        #pragma unroll 4
        for (long m = lo + y; m < hi; m += Y) {
            u32x4 u[E];
            const typename Elem<DT>::T* p = g + m * N + n;
            if (n + 8 <= N) load8<DT>(p, u);
            else load8_tail<DT>(p, (int)(N - n), u);
            float f[8];
            floats8<DT>(u, f);
            #pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += f[i];
        }
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) red[threadIdx.x][i] = v[i];
    __syncthreads();
    for (int i = threadIdx.x; i < W * 8; i += 256) {
        const long c = (long)blockIdx.x * W * 8 + i;
        if (c >= N) break;
        float s = 0.f;
        for (int k = 0; k < Y; ++k) s += red[k * W + (i >> 3)][i & 7];
        part[blockIdx.y * (long)N + c] = s;
    }
}

struct Sums { int W, chunks; long rows; unsigned gx; };
Sums sums(long M, long N) {
    Sums s;
    s.W = 1;
    while (s.W < 256 && s.W * 8 < N) s.W *= 2;
    s.gx = (unsigned)((N + s.W * 8 - 1) / (s.W * 8));
    // enough blocks for the card, at least 16 rows a lane
    const long least = 256 / s.W * 16, most = std::max<long>(1, 1024 / s.gx);
    s.rows = std::max(least, (M + most - 1) / most);
    s.chunks = (int)((M + s.rows - 1) / s.rows);
    return s;
}

// ---------------------------------------------------------------------------
// small products
// ---------------------------------------------------------------------------

struct Small {
    const void* g;
    long M, N, K;
    const uint8_t *wc, *ws, *xc, *xs;    // of the results that are wanted
    void *dx, *dw, *db;
    int dx_dt, dw_dt, db_dt;
    int dx_blocks, dw_blocks, kb;        // kb: blocks along K
};

static __device__ __forceinline__ void store_any(void* p, int dt, long i, float v) {
    if (dt == F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

// out[a, k] = sum_b g(a, b) V[b, k] for 4 values of a and 64 of k a block: 8
// lanes take 8 columns each, the 32 groups of them every 32nd b, joined in
// order. g(a, b) lies at a * ga + b * gb.
constexpr int SA = 4;
template <int DT>
static __device__ void small_product(const Small& p, long A, long B, long ga,
                                     long gb, const uint8_t* codes,
                                     const uint8_t* scales, void* out, int dt,
                                     int block) {
    const typename Elem<DT>::T* g = (const typename Elem<DT>::T*)p.g;
    __shared__ float red[32][SA][65];
    const int x = threadIdx.x & 7, y = threadIdx.x >> 3;
    const long a0 = (long)(block / p.kb) * SA, k = (long)(block % p.kb) * 64 + x * 8;
    float v[SA][8] = {};
    if (k < p.K) {
        #pragma unroll 8
        for (long b = y; b < B; b += 32) {
            const unsigned c = reinterpret_cast<const unsigned*>(codes)[
                ((size_t)(k >> 7) * B + b) * 16 + (k >> 3 & 15)];
            const unsigned byte = scales[scale_at(B, b, (int)(k >> 5))];
            float gv[SA], f[8];
            #pragma unroll
            for (int i = 0; i < SA; ++i)
                gv[i] = (float)g[min(a0 + i, A - 1) * ga + b * gb];
            values8(c, byte, f);
            #pragma unroll
            for (int i = 0; i < SA; ++i)
                #pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[i][e] = __builtin_fmaf(gv[i], f[e], v[i][e]);
        }
    }
    #pragma unroll
    for (int i = 0; i < SA; ++i)
        #pragma unroll
        for (int e = 0; e < 8; ++e) red[y][i][x * 8 + e] = v[i][e];
    __syncthreads();
    const int i = threadIdx.x >> 6, e = threadIdx.x & 63;
    const long a = a0 + i, kk = (long)(block % p.kb) * 64 + e;
    if (a >= A || kk >= p.K) return;
    float s = 0.f;
    #pragma unroll
    for (int q = 0; q < 32; ++q) s += red[q][i][e];
    store_any(out, dt, a * p.K + kk, s);
}

template <int DT>
__global__ __launch_bounds__(256)
void small_grads_kernel(const Small p) {
    int block = blockIdx.x;
    if (block < p.dx_blocks) {
        small_product<DT>(p, p.M, p.N, p.N, 1, p.wc, p.ws, p.dx, p.dx_dt, block);
        return;
    }
    block -= p.dx_blocks;
    if (block < p.dw_blocks) {
        small_product<DT>(p, p.N, p.M, 1, p.N, p.xc, p.xs, p.dw, p.dw_dt, block);
        return;
    }
    block -= p.dw_blocks;
    // 8 columns, every 32nd row a group of lanes
    __shared__ float red[32][9];
    const typename Elem<DT>::T* g = (const typename Elem<DT>::T*)p.g;
    const int x = threadIdx.x & 7, y = threadIdx.x >> 3;
    const long n = (long)block * 8 + x;
    float v = 0.f;
    if (n < p.N) {
        #pragma unroll 8
        for (long m = y; m < p.M; m += 32) v += (float)g[m * p.N + n];
    }
    red[y][x] = v;
    __syncthreads();
    if (y || n >= p.N) return;
    float s = 0.f;
    #pragma unroll
    for (int k = 0; k < 32; ++k) s += red[k][x];
    store_any(p.db, p.db_dt, n, s);
}

// ---------------------------------------------------------------------------

unsigned grid_for(long total) {
    return (unsigned)std::min<long>((total + 255) / 256, 256 * 32);
}

bool dx_in_place(const GradArgs& a) {
    return a.g_dt == BF16 && a.aligned && a.N % 32 == 0;
}
bool dw_in_place(const GradArgs& a) {
    return a.g_dt == BF16 && a.aligned && a.N % 8 == 0;
}

// One launch against five to nine of 4 us. All three gradients in us, MxKxN:
// 83x200x65 fp32 6.5 against 34, 512x512x512 bf16 21 against 44, 1024x512x512 37
// against 47 (700^3 45 against 60, but 49 without db). A lane's sum over every 32nd
// row is a chain of loads, so long sums go to the tiles: 1500x64x64 bf16 17
// against 25, 3136x64x64 34 against 24. Wider types are cut into parts first
// there: 2048x256x256 fp32 21 against 59, 4000x128x256 54 against 55.
bool small(const GradArgs& a) {
    return (double)a.M * a.N * a.K <= 0x1p28 &&
           std::max(a.M, a.N) <= (a.g_dt == BF16 ? 1536 : 2560);
}

template <bool STEPPED>
void launch_parts(const GradArgs& a, int Np, void* out, hipStream_t stream) {
    const long total = a.M * (Np / 8);
    #define MX4_G(DT) \
        hipLaunchKernelGGL((parts_kernel<DT, STEPPED>), dim3(grid_for(total)), \
                           dim3(256), 0, stream, \
                           (const typename Elem<DT>::T*)a.g, a.M, (int)a.N, Np, \
                           parts_of(a.g_dt), (u32x4*)out)
    if (a.g_dt == F32) MX4_G(F32);
    else if (a.g_dt == BF16) MX4_G(BF16);
    else MX4_G(F16);
    #undef MX4_G
}

// Both products read one set of parts, in rows: 15680x512x2048 fp32 325 us for 382
// with a set for each.
bool share_parts(const GradArgs& a) {
    return a.dx && a.dw && !dx_in_place(a) && !dw_in_place(a);
}
size_t part_bytes(const GradArgs& a, long Np) {
    return (size_t)parts_of(a.g_dt) * a.M * Np * 2;
}

// forms from 2 on ask for a tile of the input's gradient
int tile_of(int form) { return form < 2 ? -1 : form - 2; }

size_t dx_bytes(const GradArgs& a, int tile) {
    const long Np = up32(a.N);
    return up256((size_t)a.K * Np * 2)
        + (dx_in_place(a) || share_parts(a) ? 0 : up256(part_bytes(a, Np)))
        + grad_input_partial(a.M, a.K, Np / 32 * parts_of(a.g_dt), tile);
}

size_t dw_bytes(const GradArgs& a) {
    return (dw_in_place(a) || share_parts(a)
                ? 0 : up256(part_bytes(a, (a.N + 7) / 8 * 8)))
        + grad_weight_partial(a.M, a.N, a.K, parts_of(a.g_dt));
}

size_t db_bytes(const GradArgs& a) {
    return up256((size_t)sums(a.M, a.N).chunks * a.N * 4);
}

// W^T is written once as bf16 (W is small beside g, or the product large).
// `rows`: parts in rows of up32(N), where there are some.
void run_dx(const GradArgs& a, int tile, const char* rows, char* at,
            hipStream_t stream) {
    const long Np = up32(a.N);
    const int P = parts_of(a.g_dt), per = (int)(Np / 32);
    __bf16* wt = (__bf16*)at;
    at += up256((size_t)a.K * Np * 2);
    hipLaunchKernelGGL(values_t_kernel,
                       dim3((unsigned)(Np / 32), (unsigned)steps_of(a.K)),
                       dim3(256), 0, stream, a.wc, a.ws, a.N, a.K, wt);
    const size_t row = Np * 2;               // = N * 2 where g is read in place
    if (rows || dx_in_place(a)) {
        grad_input_tiles(rows ? rows : a.g, 64, row, a.M * row, P, per, wt, a.M,
                         a.K, a.dx, a.dx_dt, tile, at, stream);
        return;
    }
    char* parts = at;
    at += up256(part_bytes(a, Np));
    launch_parts<true>(a, (int)Np, parts, stream);
    grad_input_tiles(parts, (size_t)a.M * 64, 64, per * (size_t)a.M * 64, P, per,
                     wt, a.M, a.K, a.dx, a.dx_dt, tile, at, stream);
}

void run_dw(const GradArgs& a, const char* rows, char* at, hipStream_t stream) {
    const int P = parts_of(a.g_dt);
    long Np = a.N;
    const void* g = a.g;
    if (rows) {
        Np = up32(a.N);
        g = rows;
    } else if (!dw_in_place(a)) {
        Np = (a.N + 7) / 8 * 8;
        launch_parts<false>(a, (int)Np, at, stream);
        g = at;
        at += up256(part_bytes(a, Np));
    }
    grad_weight_tiles(g, Np, (size_t)a.M * Np * 2, P, a.M, a.N, a.K, a.xc, a.xs,
                      a.dw, a.dw_dt, at, stream);
}

void run_db(const GradArgs& a, char* at, hipStream_t stream) {
    const Sums s = sums(a.M, a.N);
    const dim3 grid(s.gx, (unsigned)s.chunks);
    #define MX4_S(DT) \
        hipLaunchKernelGGL((col_sum_kernel<DT>), grid, dim3(256), 0, stream, \
                           (const typename Elem<DT>::T*)a.g, a.M, (int)a.N, s.W, \
                           s.rows, (float*)at)
    if (a.g_dt == F32) MX4_S(F32);
    else if (a.g_dt == BF16) MX4_S(BF16);
    else MX4_S(F16);
    #undef MX4_S
    join((const float*)at, s.chunks, a.N, a.db, a.db_dt, stream);
}

}  // namespace

void join(const float* part, int S, long n, void* out, int dt,
          hipStream_t stream) {
    const bool many = n >= 65536;
    #define MX4_J(DT) do { \
        if (many) \
            hipLaunchKernelGGL((join_many_kernel<DT>), \
                dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, stream, part, \
                S, n, (typename Elem<DT>::T*)out); \
        else \
            hipLaunchKernelGGL((join_few_kernel<DT>), \
                dim3((unsigned)((n + 15) / 16)), dim3(256), 0, stream, part, S, \
                n, (typename Elem<DT>::T*)out); } while (0)
    if (dt == F32) MX4_J(F32);
    else if (dt == BF16) MX4_J(BF16);
    else MX4_J(F16);
    #undef MX4_J
}

size_t grads_bytes(const GradArgs& a, int form) {
    if (form < 0 ? small(a) : form == 0) return 0;
    // one after the other on the stream: the same bytes serve all
    return (share_parts(a) ? up256(part_bytes(a, up32(a.N))) : 0)
        + std::max({a.dx ? dx_bytes(a, tile_of(form)) : 0, a.dw ? dw_bytes(a) : 0,
                     a.db ? db_bytes(a) : 0});
}

void grads(const GradArgs& a, int form, void* work, hipStream_t stream) {
    if (form < 0 ? small(a) : form == 0) {
        Small p{a.g, a.M, a.N, a.K, a.wc, a.ws, a.xc, a.xs, a.dx, a.dw,
                a.db, a.dx_dt, a.dw_dt, a.db_dt, 0, 0, (int)((a.K + 63) / 64)};
        p.dx_blocks = a.dx ? (int)((a.M + SA - 1) / SA) * p.kb : 0;
        p.dw_blocks = a.dw ? (int)((a.N + SA - 1) / SA) * p.kb : 0;
        const int db = a.db ? (int)((a.N + 7) / 8) : 0;
        const dim3 grid((unsigned)(p.dx_blocks + p.dw_blocks + db));
        #define MX4_S(DT) \
            hipLaunchKernelGGL((small_grads_kernel<DT>), grid, dim3(256), 0, stream, p)
        if (a.g_dt == F32) MX4_S(F32);
        else if (a.g_dt == BF16) MX4_S(BF16);
        else MX4_S(F16);
        #undef MX4_S
        return;
    }
    char *rows = nullptr, *at = (char*)work;
    if (share_parts(a)) {
        rows = at;
        at += up256(part_bytes(a, up32(a.N)));
        launch_parts<false>(a, (int)up32(a.N), rows, stream);
    }
    if (a.dx) run_dx(a, tile_of(form), rows, at, stream);
    if (a.dw) run_dw(a, rows, at, stream);
    if (a.db) run_db(a, at, stream);
}

}  // namespace mx4
