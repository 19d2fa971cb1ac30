// dx[M,K] = g[M,N] W[N,K] on v_mfma_f32_16x16x32_bf16 (see mx4_grad.hip).
//
// A lane's operand is 16 bytes, 8 elements of the sum, and a step of 32 has
// rows of 64 bytes: the shape of the 4-bit products (mx4_tiles.hip), and the
// same machine: a ring of four buffers filled past the registers, across the
// ends of tiles, reads two rows ahead of the matrix instructions, one barrier a
// step, waits by count. g's rows are read where they are; that halves the rate
// of its copies (64 bytes of a row at a time), which a tile of 256 x 256 leaves
// time for: 764 of its 1024 cycles a step (copies of 128 bytes of a row, two steps
// at a time, changed nothing). 15680x2048 -> 512 takes 40 us, 4096^3 with W's
// layout 114 (1.2 PFLOP/s).

#include <hip/hip_runtime.h>

#include <algorithm>

#include "mx4_grad.h"

namespace mx4 {
namespace {

constexpr int S = 4;

// C is [splits][M][K] where there are several
template <int OT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 2)
void grad_input_kernel(const uint8_t* __restrict__ a, size_t a_step,
                       size_t a_row, size_t a_part, int steps, int per,
                       const uint8_t* __restrict__ b, long M, long N,
                       typename Elem<OT>::T* __restrict__ c, int mt, int nt,
                       int splits, int group) {
    constexpr int WAVES = WM * WN, R = BM + BN;
    constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
    constexpr int XQ = BM / 16 / WAVES, WQ = BN / 16 / WAVES, Q = XQ + WQ;
    static_assert(BM % (16 * WAVES) == 0 && BN % (16 * WAVES) == 0, "whole copies");
    __shared__ __attribute__((aligned(16))) uint8_t lds[S * R * 64];
    const unsigned to = lds_address(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int wm = (wave / WN) * (FM * 16), wn = (wave % WN) * (FN * 16);

    // Blocks go round the 8 dies; each has a run of tiles, `group` rows of them
    // at a time; the splits of a tile come one after the other.
    const int total = mt * nt * splits, xcd = blockIdx.x & 7;
    const int q8 = total >> 3, r8 = total & 7, stride = gridDim.x >> 3;
    const int lo = xcd * q8 + min(xcd, r8), hi = lo + q8 + (xcd < r8);
    auto place = [&](int t, long& m0, long& n0, int& s0, int& s1) {
        const int z = t % splits, u = t / splits;
        const int width = group * nt, first = u / width * group;
        const int rows = min(mt - first, group), in = u % width;
        m0 = (long)(first + in % rows) * BM;
        n0 = (long)(in / rows) * BN;
        s0 = (int)((long)steps * z / splits);
        s1 = (int)((long)steps * (z + 1) / splits);
    };

    int lt = lo + (blockIdx.x >> 3), lk = 0, lend = 0, lp = 0;
    if (lt >= hi) return;
    const uint8_t *la = a, *lb = b, *lb0 = b;
    unsigned ao[XQ], bo[WQ];
    auto aim = [&]() {
        long m0, n0;
        place(lt, m0, n0, lk, lend);
        const int lasta = (int)min((long)BM, M - m0) - 1;
        const int lastb = (int)min((long)BN, N - n0) - 1;
        lp = lk % per;                            // step of this part
        la = a + lk / per * a_part + lp * a_step + m0 * a_row;
        lb0 = b + n0 * 64;
        lb = lb0 + (size_t)lp * N * 64;
        #pragma unroll
        for (int q = 0; q < XQ; ++q) {
            const int r = (q * WAVES + wave) * 16 + (lane >> 2);
            ao[q] = (unsigned)min(r, lasta) * (unsigned)a_row
                + ((lane & 3) ^ x_key(r)) * 16;
        }
        #pragma unroll
        for (int q = 0; q < WQ; ++q) {
            const int r = (q * WAVES + wave) * 16 + (lane >> 2);
            bo[q] = min(r, lastb) * 64 + ((lane & 3) ^ w_key<FN>(r)) * 16;
        }
    };
    const size_t next_part = a_part - per * a_step;
    bool more = true;
    auto send = [&](int buf, int q) {
        if (q < XQ)
            copy16_to_lds(la, ao[q], to + buf * (R * 64) + (q * WAVES + wave) * 1024);
        else
            copy16_to_lds(lb, bo[q - XQ], to + buf * (R * 64) + BM * 64
                                              + ((q - XQ) * WAVES + wave) * 1024);
    };
    // (behind the last step the same bytes are sent again: the waits count)
    auto sent = [&]() {
        if (!more) return;
        la += a_step, lb += (size_t)N * 64;
        if (++lp == per) lp = 0, lb = lb0, la += next_part;
        if (++lk == lend) {
            more = lt + stride < hi;
            if (more) lt += stride;
            aim();
        }
    };
    aim();
    #pragma unroll
    for (int i = 0; i < S - 1; ++i) {
        if (i) sent();
        #pragma unroll
        for (int q = 0; q < Q; ++q) send(i, q);
    }

    const int xr = wm + r16, wr = wn + (r16 >> 2) * (4 * FN) + (r16 & 3);
    const int xp = xr * 64 + ((g ^ x_key(xr)) << 4);
    const int wp = (BM + wr) * 64 + ((g ^ w_key<FN>(wr)) << 4);
    int buf = 0;
    bf16x8 w[FN], x[FM];
    auto begin = [&](int at) {
        const uint8_t* p = lds + at * (R * 64);
        #pragma unroll
        for (int j = 0; j < FN; ++j)
            w[j] = *reinterpret_cast<const bf16x8*>(p + wp + j * 256);
        x[0] = *reinterpret_cast<const bf16x8*>(p + xp);
        if (FM > 1) x[1] = *reinterpret_cast<const bf16x8*>(p + xp + 1024);
    };
    wait_copies<0>();
    __syncthreads();
    begin(0);
    for (int t = lo + (blockIdx.x >> 3); t < hi; t += stride) {
        long m0, n0;
        int s0, s1;
        place(t, m0, n0, s0, s1);
        f32x4 acc[FM][FN];
        #pragma unroll
        for (int i = 0; i < FM; ++i)
            #pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};
        for (int k = s0; k < s1; ++k) {
            // the bytes of the step behind this one have arrived, and every
            // wave is done with the buffer of the step before
            wait_copies<(S - 3) * Q>();
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            const int free = buf == 0 ? S - 1 : buf - 1;
            const uint8_t* p = lds + buf * (R * 64);
            buf = buf == S - 1 ? 0 : buf + 1;
            sent();
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (i + 2 < FM)
                    x[i + 2] = *reinterpret_cast<const bf16x8*>(p + xp + (i + 2) * 1024);
                #pragma unroll
                for (int q = i * Q / FM; q < (i + 1) * Q / FM; ++q) send(free, q);
                #pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        w[j], x[i], acc[i][j], 0, 0, 0);
            }
            begin(buf);
            #pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (i + 2 < FM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                if (i == FM - 1) __builtin_amdgcn_sched_group_barrier(
                    0x100, FN + (FM > 1 ? 2 : 1), 0);
                __builtin_amdgcn_sched_group_barrier(0x8, FN, 0);
            }
        }
        const float none[4 * FN] = {};
        store_rows<OT, FM, FN>(acc, c + (splits > 1 ? (size_t)(t % splits) * M * N : 0),
                               M, N, m0 + wm + r16, n0 + wn + g * (4 * FN), none);
    }
    wait_copies<0>();      // no copy is under way when LDS is given up
}

// The tile that ends first: rounds over the blocks that fit, times the cycles of
// a step (of all blocks on a unit). 15680x512 (sum 2048): 256 x 256 50 us, 256 x
// 128 40, 128 x 128 43. Few columns: 256 x 64.
struct Plan { int bm, bn, slots, splits; };
Plan plan(long M, long K, long steps, int tile) {
    static const struct { int bm, bn, slots, cycles; } T[TILES] = {
        {256, 256, 256, 1260}, {256, 128, 256, 780}, {128, 128, 512, 1380},
        {256, 64, 512, 1000}};
    Plan p{};
    double best = 0;
    for (int i = 0; i < TILES; ++i) {
        if (tile >= 0 && i != tile) continue;
        const auto& t = T[i];
        const long have = ((M + t.bm - 1) / t.bm) * ((K + t.bn - 1) / t.bn);
        const double cost = (double)((have + t.slots - 1) / t.slots) * t.cycles;
        if (p.bm && cost >= best) continue;
        best = cost;
        p = {t.bm, t.bn, t.slots, 1};
        // a long sum with few tiles is split, at least 8 steps each
        if (have * 4 <= t.slots)
            p.splits = (int)std::max<long>(1, std::min(t.slots / have, steps / 8));
    }
    return p;
}

}  // namespace

size_t grad_input_partial(long M, long K, long steps, int tile) {
    const int s = plan(M, K, steps, tile).splits;
    return s > 1 ? up256((size_t)s * M * K * 4) : 0;
}

void grad_input_tiles(const void* a, size_t a_step, size_t a_row, size_t a_part,
                      int parts, int per, const void* b, long M, long K,
                      void* c, int dt, int tile, void* partial,
                      hipStream_t stream) {
    const int steps = per * parts;
    const Plan p = plan(M, K, steps, tile);
    const int mt = (int)((M + p.bm - 1) / p.bm), nt = (int)((K + p.bn - 1) / p.bn);
    void* out = p.splits > 1 ? partial : c;
    const int odt = p.splits > 1 ? F32 : dt;
    const int total = mt * nt * p.splits;
    #define MX4_G(OT, BM, BN, WM, WN) \
        hipLaunchKernelGGL((grad_input_kernel<OT, BM, BN, WM, WN>), \
            dim3(std::min((total + 7) / 8 * 8, p.slots)), \
            dim3(64 * WM * WN), 0, stream, (const uint8_t*)a, a_step, a_row, \
            a_part, steps, per, (const uint8_t*)b, M, K, (typename Elem<OT>::T*)out, mt, \
            nt, p.splits, 4)
    #define MX4_T(OT) do { \
        if (p.bn == 256) MX4_G(OT, 256, 256, 2, 4); \
        else if (p.bm == 256 && p.bn == 128) MX4_G(OT, 256, 128, 4, 2); \
        else if (p.bn == 128) MX4_G(OT, 128, 128, 2, 2); \
        else MX4_G(OT, 256, 64, 4, 1); } while (0)
    if (odt == F32) MX4_T(F32);
    else if (odt == BF16) MX4_T(BF16);
    else MX4_T(F16);
    #undef MX4_T
    #undef MX4_G
    if (p.splits > 1) join((const float*)partial, p.splits, M * K, c, dt, stream);
}

}  // namespace mx4
