// Shared by the MX4 kernels: types, the block rounding, the launchers.
//
// MX4 (OCP Microscaling Formats v1.0, MXFP4): 32 consecutive elements of a
// row share a power-of-two scale, each element is one of
// {0, .5, 1, 1.5, 2, 3, 4, 6} with a sign:
//   E = clamp(floor(log2 max|x|) - 2, -127, 127), byte = E + 127
//   q = x * 2^-E to the nearest value, ties to the even code, 6 at most.
// A block with a NaN or an infinity has byte 255 and reads as NaN.
//
// Storage of [R, K], for the matrix cores' reads: rows are padded with zeros to
// Kp, a multiple of 128 elements (one step of v_mfma_scale_f32_16x16x128), and
//   codes  [Kp/128][R][64]: a step's 64 bytes of all rows in one piece, so that
//          any run of rows is one run of memory for a step;
//   scales [up(Kp/512)][R][16]: of four steps, byte 4*g + s is the scale of
//          block g of step s, so that lane group g has its four in one word and
//          the instruction picks the byte of the step.
// Codes: low nibble first. Scales of the padding are 0 as well.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace mx4 {

enum DType : int { F32 = 0, BF16 = 1, F16 = 2 };

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

template <int DT> struct Elem;
template <> struct Elem<F32> { using T = float; };
template <> struct Elem<BF16> { using T = __bf16; };
template <> struct Elem<F16> { using T = _Float16; };

// one rounding, to nearest even
template <int DT>
static __device__ __forceinline__ typename Elem<DT>::T from_f32(float v) {
    return (typename Elem<DT>::T)v;
}

// 2^(byte-127) as a float; 2^-127 lies below the normal numbers, and byte 255
// gives an infinity.
static __device__ __forceinline__ float scale_f32(unsigned byte) {
    return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// max|x| of packed 16-bit floats by their bits (the order of the absolute
// bits is the order of the values, infinities and NaN on top)
static __device__ __forceinline__ u16x2 absmax16(u16x2 m, unsigned w) {
    w &= 0x7fff7fffu;
    return __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w));
}

template <int DT>
static __device__ __forceinline__ unsigned absmax_bits(const u32x4* u, int n4) {
    if constexpr (DT == F32) {
        unsigned m = 0;
        #pragma unroll
        for (int i = 0; i < n4; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                m = max(m, u[i][j] & 0x7fffffffu);
        return m;
    } else {
        u16x2 m = {0, 0};
        #pragma unroll
        for (int i = 0; i < n4; ++i)
            #pragma unroll
            for (int j = 0; j < 4; ++j) m = absmax16(m, u[i][j]);
        return max((unsigned)m.x, (unsigned)m.y);
    }
}

// scale byte of a block from the bits of its absolute maximum
template <int DT>
static __device__ __forceinline__ unsigned scale_byte(unsigned bits) {
    unsigned e;
    if constexpr (DT == F32) {
        if (bits >= 0x7f800000u) return 255u;
        e = bits >> 23;
    } else if constexpr (DT == BF16) {
        if (bits >= 0x7f80u) return 255u;
        e = bits >> 7;
    } else {
        if (bits >= 0x7c00u) return 255u;
        // exact in fp32, where fp16's subnormal numbers are normal
        e = __float_as_uint((float)__builtin_bit_cast(
                _Float16, (unsigned short)bits)) >> 23;
    }
    return e > 2u ? e - 2u : 0u;   // (e - 127) - 2 + 127, at least 0
}

// (by value: a bit cast of a vector's element in place takes the first one)
static __device__ __forceinline__ bf16x2 as_bf16x2(unsigned w) {
    return __builtin_bit_cast(bf16x2, w);
}
static __device__ __forceinline__ f16x2 as_f16x2(unsigned w) {
    return __builtin_bit_cast(f16x2, w);
}

// 8 elements (one 16-byte word of 16-bit floats, two of fp32) to 8 codes.
// The conversion instructions divide by the scale, round to nearest even and
// saturate at 6; checked value by value, subnormal scale included.
template <int DT>
static __device__ __forceinline__ unsigned codes8(const u32x4* u, float s) {
    unsigned r = 0;
    if constexpr (DT == F32) {
        const u32x4 a = u[0], b = u[1];
        #define MX4_F(i) __uint_as_float(i)
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, MX4_F(a.x), MX4_F(a.y), s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, MX4_F(a.z), MX4_F(a.w), s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, MX4_F(b.x), MX4_F(b.y), s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, MX4_F(b.z), MX4_F(b.w), s, 3);
        #undef MX4_F
    } else if constexpr (DT == BF16) {
        const u32x4 a = u[0];
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16x2(a.x), s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16x2(a.y), s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16x2(a.z), s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_bf16x2(a.w), s, 3);
    } else {
        const u32x4 a = u[0];
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_f16x2(a.x), s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_f16x2(a.y), s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_f16x2(a.z), s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_f16x2(a.w), s, 3);
    }
    return r;
}

// 8 elements at p, which need not start on 16 bytes: the memory pipe takes any
// address in one load. With this and store_piece, fp32 5000x777->777 takes 21 us;
// 41 with single elements.
template <int DT>
static __device__ __forceinline__ void load8(const typename Elem<DT>::T* p,
                                             u32x4* u) {
    struct __attribute__((packed, aligned(sizeof(*p)))) Any {
        u32x4 v[DT == F32 ? 2 : 1];
    };
    const Any a = *reinterpret_cast<const Any*>(p);
    u[0] = a.v[0];
    if constexpr (DT == F32) u[1] = a.v[1];
}

// n elements at p, eight at most, the rest zero: one load where there are eight,
// pieces of 4, 2 and 1 where the row ends (777x333->1001 fp16 8.3 us; 9.3 with single
// elements).
template <int DT>
static __device__ __forceinline__ void load8_tail(
        const typename Elem<DT>::T* p, int n, u32x4* u) {
    constexpr int W = DT == F32 ? 2 : 1;
    if (n >= 8) {
        load8<DT>(p, u);
        return;
    }
    #pragma unroll
    for (int i = 0; i < W; ++i) u[i] = (u32x4){0, 0, 0, 0};
    if (n <= 0) return;
    if constexpr (DT == F32) {
        struct __attribute__((packed, aligned(4))) Four { u32x4 v; };
        const unsigned* q = reinterpret_cast<const unsigned*>(p);
        unsigned r[3] = {0, 0, 0};
        if (n & 4) u[0] = reinterpret_cast<const Four*>(q)->v;
        q += n & 4;
        #pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < (n & 3)) r[i] = q[i];
        const u32x4 v = {r[0], r[1], r[2], 0};
        if (n & 4) u[1] = v;
        else u[0] = v;
    } else {
        struct __attribute__((packed, aligned(2))) Four { u32x2 v; };
        struct __attribute__((packed, aligned(2))) Two { unsigned v; };
        const unsigned short* q = reinterpret_cast<const unsigned short*>(p);
        u32x2 four = {0, 0};
        unsigned two = 0, one = 0;
        if (n & 4) four = reinterpret_cast<const Four*>(q)->v;
        q += n & 4;
        if (n & 2) two = reinterpret_cast<const Two*>(q)->v;
        q += n & 2;
        if (n & 1) one = *q;
        const unsigned lo = n & 2 ? two : one, hi = n & 2 ? one : 0u;
        u[0] = n & 4 ? (u32x4){four.x, four.y, lo, hi} : (u32x4){lo, hi, 0, 0};
    }
}

// W consecutive elements, 8 or 16 bytes of them at a time
template <class T, int W>
union Piece {
    static constexpr int B = W * sizeof(T) % 16 ? 8 : 16;   // bytes a store
    typedef unsigned Word __attribute__((ext_vector_type(B / 4)));
    T v[W];
    Word u[W * sizeof(T) / B];
};
// Whole where n >= W elements are left for it, wherever q points. STREAM: past
// the caches, for rows that are written in one go (where a row is written in
// parts, the L2 has to gather them: 62720x1024->256 took 42 us for 38 with it).
template <bool STREAM = false, class T, int W>
static __device__ __forceinline__ void store_piece(T* q, const Piece<T, W>& o,
                                                   long n) {
    using P = Piece<T, W>;
    typedef typename P::Word Loose __attribute__((aligned(sizeof(T))));
    if (n >= W) {
        Loose* to = reinterpret_cast<Loose*>(q);
        #pragma unroll
        for (int i = 0; i < (int)(W * sizeof(T)) / P::B; ++i) {
            if constexpr (STREAM) __builtin_nontemporal_store(o.u[i], to + i);
            else to[i] = o.u[i];
        }
    } else {
        #pragma unroll
        for (int e = 0; e < W; ++e)
            if (e < n) q[e] = o.v[e];
    }
}

constexpr int STEP = 128;              // elements of a step

static inline __host__ __device__ long steps_of(long K) { return (K + 127) / 128; }
static inline __host__ __device__ long chunks_of(long K) { return (K + 511) / 512; }
static inline size_t code_bytes(long R, long K) { return (size_t)steps_of(K) * R * 64; }
static inline size_t scale_bytes(long R, long K) { return (size_t)chunks_of(K) * R * 16; }

// where block b (of 32) of a row has its scale
static __device__ __forceinline__ size_t scale_at(long R, long row, int b) {
    return ((size_t)(b >> 4) * R + row) * 16 + (b & 3) * 4 + (b >> 2 & 3);
}

// Everything below takes strides in elements and runs on `stream`. Sizes are
// checked by callers.

void quantize(const void* x, int dt, long rows, long K, long ldx,
              uint8_t* codes, uint8_t* scales, hipStream_t stream);

// two matrices of K columns in one launch
void quantize_two(const void* x, int dt, long rows, long ldx, uint8_t* codes,
                  uint8_t* scales, const void* x2, int dt2, long rows2,
                  long ldx2, uint8_t* codes2, uint8_t* scales2, long K,
                  hipStream_t stream);

void dequantize(const uint8_t* codes, const uint8_t* scales, long rows,
                long K, void* out, int dt, hipStream_t stream);

// Forms of the product; linear_form() and linear_q_form() choose. Each is right
// for every size.
enum Form : int {
    ROWS16 = 0,       // 16 x 16 or 32 of y a block, x rounded by each block
    ROWS32 = 1,       // 32 x 32, the same
    ROUNDING = 2,     // tiles of 64 rows, x rounded on its way into LDS
    HELD16 = 3,       // x rounded before; then the same from 4-bit rows,
    HELD32 = 4,
    TILES128 = 5,     // or tiles of them
    TILES256 = 6,
    FORMS = 7
};

// y[M,N] = Q(x) W^T + bias
int linear_form(long M, long K, long N);
size_t linear_bytes(int form, long M, long K);        // of workspace
void linear(const void* x, int dt, long M, long K, long ldx,
            const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
            int bias_dt, void* y, int form, void* work, hipStream_t stream);

// the same from rows that are held in 4 bits already
int linear_q_form(long M, long K, long N);
void linear_q(const uint8_t* xc, const uint8_t* xs, long M, long K,
              const uint8_t* wc, const uint8_t* ws, long N, const void* bias,
              int bias_dt, void* y, int dt, int form, hipStream_t stream);

// The gradients that are wanted of the product: dx[M,K] = g[M,N] W[N,K],
// dw[N,K] = g^T X[M,K], db[N] = sum_m g; none of M, N, K is 0. `aligned`: g starts
// on 16 bytes. Form 0 is the one of small products, 1 that of large ones, 2 to 5 are
// the same with a certain tile for dx, -1 chooses.
struct GradArgs {
    const void* g;
    int g_dt;
    bool aligned;
    long M, N, K;
    const uint8_t *wc, *ws, *xc, *xs;
    void *dx, *dw, *db;                  // null where not wanted
    int dx_dt, dw_dt, db_dt;
};
constexpr int GRAD_FORMS = 6;
size_t grads_bytes(const GradArgs& a, int form);      // of workspace
void grads(const GradArgs& a, int form, void* work, hipStream_t stream);

}  // namespace mx4
