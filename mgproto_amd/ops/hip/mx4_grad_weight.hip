// dw[N,K] = g[M,N]^T X[M,K] on v_mfma_f32_16x16x32_bf16 (see mx4_grad.hip).
//
// The sum runs over rows, so both operands are wanted across their rows. g's
// rows go into LDS as they are, past the registers; X's codes, a quarter of
// that, go there as codes and are written beside as bf16 (every value is exact
// in it) two steps ahead. ds_read_b64_tr_b16 then gives a lane four rows of one
// column: two of them are its operand, in the same order on both sides. So
// neither operand is ever turned in memory.
//
// 32-byte pieces c of row m lie at c ^ key(m): the 16 rows that one read takes
// fall on all banks twice, which is what 512 bytes need.
//
// With few results the sum is split over blocks and joined in order.
//
// The reads across rows take 8 bytes a lane and so as many cycles as the matrix
// instructions they feed; 4096^3 takes 147 us (0.93 PFLOP/s), 15680x512x2048 49 and
// its join 13.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_grad.h"

namespace mx4 {
namespace {

constexpr int S = 5;            // buffers of g and of codes
constexpr int XS = 3;           // of X as bf16
constexpr int ROWS = 32;        // of a step

typedef short s16x4 __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ bf16x8 read_across(const uint8_t* p,
                                                     const uint8_t* q) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(uint32_t)(uintptr_t)p);
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(uint32_t)(uintptr_t)q);
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(
        a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// rows of BYTES: at most as many places as there are pieces
template <int BYTES> static __device__ __forceinline__ int row_key(int m) {
    if constexpr (BYTES >= 256) return (m & 3) | (m >> 3 & 1) << 2;
    else return (m >> 1 & 1) | (m >> 3 & 1) << 1;       // rows of 128
}

template <int OT, int TN, int TK, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2)
void grad_weight_kernel(const uint8_t* __restrict__ gv, long row, size_t part,
                        int parts, long M, long N, long K,
                        const uint8_t* __restrict__ xc,
                        const uint8_t* __restrict__ xs,
                        typename Elem<OT>::T* __restrict__ c, int nt, int kt,
                        int splits) {
    using T = typename Elem<OT>::T;
    constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    constexpr int FM = TN / WM / 16, FN = TK / WN / 16;
    constexpr int GB = TN * 2, XB = TK * 2;              // bytes of a row
    constexpr int GC = ROWS * GB / 1024 / WAVES;         // copies a step
    constexpr int XSTEPS = TK > 128 ? TK / 128 : 1;      // 128s of the codes
    constexpr int XC = 2 * XSTEPS + 1;                   // copies: codes, scales
    constexpr int XQ = (XC + WAVES - 1) / WAVES;
    constexpr int PER = GC + XQ;
    constexpr int STAGE = ROWS * GB + XC * 1024;
    static_assert(ROWS * GB % (1024 * WAVES) == 0 &&
                  ROWS * TK / 8 % THREADS == 0, "whole copies, whole words");
    __shared__ __attribute__((aligned(16))) uint8_t lds[S * STAGE + XS * ROWS * XB];
    uint8_t* const xl = lds + S * STAGE;
    const unsigned to = lds_address(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int wm = (wave / WN) * (FM * 16), wn = (wave % WN) * (FN * 16);

    // the splits of neighbouring tiles together on a die: they read the same g
    const int total = nt * kt * splits, xcd = blockIdx.x & 7;
    const int q8 = total >> 3, r8 = total & 7;
    const int t = xcd * q8 + min(xcd, r8) + (blockIdx.x >> 3);
    const int z = t / (nt * kt), u = t % (nt * kt);
    const long n0 = (long)(u / kt) * TN, k0 = (long)(u % kt) * TK;
    const int per = (int)((M + ROWS - 1) / ROWS);        // steps of a part
    const int s0 = (int)((long)per * parts * z / splits);
    const int s1 = (int)((long)per * parts * (z + 1) / splits);

    // g: pieces of 16 bytes; behind the last column the last piece again
    constexpr int PIECES = GB / 16;
    const int lastp = (int)min((long)PIECES, (N + 7) / 8 - n0 / 8) - 1;
    int gr[GC], gp[GC];
    #pragma unroll
    for (int q = 0; q < GC; ++q) {
        const int at = (q * WAVES + wave) * 64 + lane;
        gr[q] = at / PIECES;
        const int p = at % PIECES;
        gp[q] = min(((p >> 1) ^ row_key<GB>(gr[q])) << 1 | (p & 1), lastp) * 16;
    }
    int ls = s0, lp = s0 / per, lm = s0 % per;           // step, part, of it
    auto send = [&](int buf) {
        const long m0 = (long)lm * ROWS;
        const int last = (int)min((long)ROWS, M - m0) - 1;
        const uint8_t* base = gv + lp * part + (m0 * row + n0) * 2;
        #pragma unroll
        for (int q = 0; q < GC; ++q)
            copy16_to_lds(base, (unsigned)(min(gr[q], last) * row * 2) + gp[q],
                          to + buf * STAGE + (q * WAVES + wave) * 1024);
        #pragma unroll
        for (int q = 0; q < XQ; ++q) {
            const int call = min(q * WAVES + wave, XC - 1);
            const unsigned l = to + buf * STAGE + ROWS * GB + call * 1024;
            if (call < XC - 1)       // 16 rows of 64 bytes
                copy16_to_lds(xc + ((size_t)(min((int)(k0 >> 7) + (call >> 1),
                                                 (int)steps_of(K) - 1)) * M + m0) * 64,
                              min((call & 1) * 16 + (lane >> 2), last) * 64
                                  + (lane & 3) * 16, l);
            else                     // 32 rows of 16 bytes, twice
                copy16_to_lds(xs + ((size_t)(k0 >> 9) * M + m0) * 16,
                              min(lane & 31, last) * 16, l);
        }
    };
    auto sent = [&]() {              // behind the end the last step again
        if (ls + 1 >= s1) return;
        ++ls;
        if (++lm == per) lm = 0, ++lp;
    };

    // the codes of a step as bf16: 8 of them a thread at a time, fetched before
    // the matrix instructions of a step and written behind them
    constexpr int WORDS = ROWS * TK / 8 / THREADS;
    unsigned code[WORDS], byte[WORDS];
    auto fetch = [&](int buf) {
        const uint8_t* cl = lds + buf * STAGE + ROWS * GB;
        #pragma unroll
        for (int q = 0; q < WORDS; ++q) {
            const int w = q * THREADS + threadIdx.x;
            const int m = w / (TK / 8), k8 = w % (TK / 8);   // row, 8 columns
            const int k = (int)(k0 & 127) + k8 * 8;          // from a 128 on
            const int b = (((int)k0 + k8 * 8) & 511) >> 5;
            code[q] = *reinterpret_cast<const unsigned*>(
                cl + (k >> 7) * 2048 + m * 64 + (k & 127) / 2);
            byte[q] = cl[(XC - 1) * 1024 + m * 16 + (b & 3) * 4 + (b >> 2)];
        }
    };
    auto expand = [&](int to_x, long m0) {
        const bool tail = m0 + ROWS > M;
        #pragma unroll
        for (int q = 0; q < WORDS; ++q) {
            const int w = q * THREADS + threadIdx.x;
            const int m = w / (TK / 8), k8 = w % (TK / 8);
            const float s = scale_f32(byte[q]);
            const unsigned c = code[q];
            u32x4 v;
            v.x = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
            v.y = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
            v.z = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
            v.w = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
            if (tail && m0 + m >= M) v = (u32x4){0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(
                xl + to_x * (ROWS * XB) + m * XB
                + (((k8 >> 1) ^ row_key<XB>(m)) << 5) + (k8 & 1) * 16) = v;
        }
    };

    // Where this lane reads: rows g*8 + r16/4 (and 4 more, which have the same
    // key), columns 4 (r16 & 3) of a fragment, whose 32 bytes are one piece.
    const int row0 = g * 8 + (r16 >> 2), in = (r16 & 3) * 8;
    int ga[FM], xa[FN];
    #pragma unroll
    for (int i = 0; i < FM; ++i)
        ga[i] = row0 * GB + (((wm / 16 + i) ^ row_key<GB>(row0)) << 5) + in;
    #pragma unroll
    for (int j = 0; j < FN; ++j)
        xa[j] = row0 * XB + (((wn / 16 + j) ^ row_key<XB>(row0)) << 5) + in;
    auto g_frag = [&](const uint8_t* p, int i) {
        return read_across(p + ga[i], p + ga[i] + 4 * GB);
    };
    auto x_frag = [&](const uint8_t* p, int j) {
        return read_across(p + xa[j], p + xa[j] + 4 * XB);
    };

    f32x4 acc[FM][FN];
    #pragma unroll
    for (int i = 0; i < FM; ++i)
        #pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};

    // rows of g that are not there, in the buffer of step `m` of a part
    auto clear_tail = [&](int buf, int m) {
        if ((long)(m + 1) * ROWS <= M) return;
        uint8_t* gl = lds + buf * STAGE;
        const int have = (int)(M - (long)m * ROWS);
        for (int i = have * (GB / 16) + threadIdx.x; i < ROWS * (GB / 16);
             i += THREADS)
            reinterpret_cast<u32x4*>(gl)[i] = (u32x4){0, 0, 0, 0};
        __syncthreads();
    };
    bf16x8 b[FN], av[FM];
    // the first reads of a step, made while the step before still computes
    auto begin = [&](int buf, int xbuf) {
        const uint8_t* gl = lds + buf * STAGE;
        const uint8_t* xp = xl + xbuf * (ROWS * XB);
        #pragma unroll
        for (int j = 0; j < FN; ++j)
            b[j] = x_frag(xp, j);
        #pragma unroll
        for (int i = 0; i < 2; ++i)
            av[i] = g_frag(gl, i);
    };

    auto turn = [](int v, int n) { return v == n - 1 ? 0 : v + 1; };
    #pragma unroll
    for (int i = 0; i < S - 1; ++i) {
        if (i) sent();
        send(i);
    }
    int cm = s0 % per;                   // step of its part
    wait_copies<0>();
    __syncthreads();
    fetch(0);
    expand(0, (long)cm * ROWS);
    fetch(1);
    expand(1, (long)turn(cm, per) * ROWS);
    clear_tail(0, cm);
    __syncthreads();
    begin(0, 0);
    int buf = 0, xbuf = 0;
    for (int s = s0; s < s1; ++s) {
        // The copies of the two steps behind this one have arrived, the next
        // step's X is written, and every wave is done with the buffers of the
        // step before.
        wait_copies<(S - 4) * PER>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint8_t* gl = lds + buf * STAGE;
        const int free = buf == 0 ? S - 1 : buf - 1;
        buf = turn(buf, S), xbuf = turn(xbuf, XS), cm = turn(cm, per);
        clear_tail(buf, cm);
        sent();
        send(free);
        // X of the step after the next (behind the end it is not read); reads
        // two fragments ahead of the matrix instructions
        fetch(turn(buf, S));
        #pragma unroll
        for (int i = 0; i < FM; ++i) {
            if (i + 2 < FM)
                av[i + 2] = g_frag(gl, i + 2);
            #pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    b[j], av[i], acc[i][j], 0, 0, 0);
        }
        begin(buf, xbuf);
        expand(turn(xbuf, XS), (long)turn(cm, per) * ROWS);
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * WORDS, 0);
        #pragma unroll
        for (int i = 0; i < FM; ++i) {
            if (i + 2 < FM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            if (i == FM - 1) __builtin_amdgcn_sched_group_barrier(0x100, 2 * FN + 4, 0);
            __builtin_amdgcn_sched_group_barrier(0x8, FN, 0);
        }
    }
    wait_copies<0>();      // no copy is under way when LDS is given up

    // a lane holds 4 consecutive columns of row n of each fragment
    T* out = c + (splits > 1 ? (size_t)z * N * K : 0);
    #pragma unroll
    for (int i = 0; i < FM; ++i) {
        const long n = n0 + wm + i * 16 + r16;
        if (n >= N) continue;
        #pragma unroll
        for (int j = 0; j < FN; ++j) {
            const long k = k0 + wn + j * 16 + g * 4;
            Piece<T, 4> o;
            #pragma unroll
            for (int r = 0; r < 4; ++r) o.v[r] = from_f32<OT>(acc[i][j][r]);
            store_piece(out + n * K + k, o, K - k);
        }
    }
}

struct Plan { int tn, tk, splits; };
Plan plan(long M, long N, long K, int parts) {
    Plan p;
    if (N <= 64 || K <= 64) p = {64, 64, 1};
    else if (N > 128 && K > 128) p = {256, 256, 1};
    else p = {128, 128, 1};
    const long have = ((N + p.tn - 1) / p.tn) * ((K + p.tk - 1) / p.tk);
    const long steps = (M + ROWS - 1) / ROWS * parts;
    const long want = p.tn == 256 ? 256 : 512;
    p.splits = (int)std::max<long>(1, std::min(want / have, steps / 8));
    return p;
}

}  // namespace

size_t grad_weight_partial(long M, long N, long K, int parts) {
    const int s = plan(M, N, K, parts).splits;
    return s > 1 ? up256((size_t)s * N * K * 4) : 0;
}

void grad_weight_tiles(const void* g, long row, size_t part, int parts, long M,
                       long N, long K, const uint8_t* xc, const uint8_t* xs,
                       void* c, int dt, void* partial, hipStream_t stream) {
    const Plan p = plan(M, N, K, parts);
    const int nt = (int)((N + p.tn - 1) / p.tn), kt = (int)((K + p.tk - 1) / p.tk);
    void* out = p.splits > 1 ? partial : c;
    const int odt = p.splits > 1 ? F32 : dt;
    #define MX4_G(OT, TN, TK, WM, WN) \
        hipLaunchKernelGGL((grad_weight_kernel<OT, TN, TK, WM, WN>), \
            dim3((unsigned)(nt * kt * p.splits)), dim3(64 * WM * WN), 0, stream, \
            (const uint8_t*)g, row, part, parts, M, N, K, xc, xs, \
            (typename Elem<OT>::T*)out, nt, kt, p.splits)
    #define MX4_T(OT) do { \
        if (p.tn == 256) MX4_G(OT, 256, 256, 2, 4); \
        else if (p.tn == 128) MX4_G(OT, 128, 128, 2, 2); \
        else MX4_G(OT, 64, 64, 2, 2); } while (0)
    if (odt == F32) MX4_T(F32);
    else if (odt == BF16) MX4_T(BF16);
    else MX4_T(F16);
    #undef MX4_T
    #undef MX4_G
    if (p.splits > 1) join((const float*)partial, p.splits, N * K, c, dt, stream);
}

}  // namespace mx4
