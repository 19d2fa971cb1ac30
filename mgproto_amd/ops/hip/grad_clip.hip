// Global gradient norm and clipping over many tensors.
//
//   N = (sum_t sum_i |g|^p)^(1/p), p = 1, 2 or infinity
//   g <- g * min(1, max_norm / (N + 1e-6))
//
// Bound by memory: the list is read for the norm, then read and written once
// to be scaled. Sums are held in 64 bits: squares of large fp32 values leave
// the range of fp32, and at one 64-bit multiply-add an element the vector
// units are far from their limit.
//
// The list travels in the kernels' own arguments, up to TENSORS of them a
// launch: nothing is uploaded, so a captured graph holds everything it needs
// and a call never waits for the host. Every sum has a fixed order.

#include <hip/hip_runtime.h>

#include "grad_clip.h"

namespace gradclip {
namespace {

constexpr int F32 = 0, BF16 = 1;         // 2 = fp16
constexpr int TENSORS = 112;             // the arguments end below 4 KB
constexpr int CHUNK = 8192;              // elements a block takes at a time
constexpr int BLOCKS = 2048;             // of a launch, at most

struct Batch {
    const void* src[TENSORS];
    void* dst[TENSORS];
    int64_t n[TENSORS];
    int first[TENSORS + 1];              // first chunk of each tensor
    uint8_t src_dt[TENSORS], dst_dt[TENSORS];
    int count;
};
static_assert(sizeof(Batch) <= 4000, "kernel arguments");

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ float lo16(unsigned w, int dt) {
    return dt == BF16 ? __uint_as_float(w << 16)
                      : (float)__builtin_bit_cast(_Float16, (unsigned short)w);
}
static __device__ __forceinline__ float hi16(unsigned w, int dt) {
    return dt == BF16 ? __uint_as_float(w & 0xffff0000u)
                      : (float)__builtin_bit_cast(_Float16,
                                                  (unsigned short)(w >> 16));
}
static __device__ __forceinline__ float load1(const void* p, int64_t i, int dt) {
    if (dt == F32) return reinterpret_cast<const float*>(p)[i];
    return lo16(reinterpret_cast<const unsigned short*>(p)[i], dt);
}
static __device__ __forceinline__ void store1(void* p, int64_t i, int dt, float v) {
    if (dt == F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}

template <int KIND>
static __device__ __forceinline__ void add(double& acc, float v) {
    if constexpr (KIND == L2) acc = __builtin_fma((double)v, (double)v, acc);
    else if constexpr (KIND == L1) acc += (double)__builtin_fabsf(v);
    else {
        // NaN stays: a comparison with it is false both ways
        const double a = (double)__builtin_fabsf(v);
        acc = a > acc || a != a ? a : acc;
    }
}
template <int KIND>
static __device__ __forceinline__ double both(double a, double b) {
    if constexpr (KIND == LINF) return b > a || b != b ? b : a;
    else return a + b;
}

static __device__ __forceinline__ int tensor_of(const Batch& b, int chunk) {
    int lo = 0, hi = b.count - 1;        // the last with first <= chunk
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int KIND>
static __device__ double block_total(double v) {
    __shared__ double red[4];
    #pragma unroll
    for (int o = 32; o; o >>= 1) v = both<KIND>(v, __shfl_xor(v, o));
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    return both<KIND>(both<KIND>(red[0], red[1]), both<KIND>(red[2], red[3]));
}

template <int KIND>
__global__ __launch_bounds__(256)
void norm_kernel(const Batch b, double* __restrict__ part) {
    double acc[4] = {0, 0, 0, 0};
    const int chunks = b.first[b.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = tensor_of(b, c);
        const int dt = b.src_dt[t];
        const int64_t at = (int64_t)(c - b.first[t]) * CHUNK;
        const int n = (int)min((int64_t)CHUNK, b.n[t] - at);
        const char* p = (const char*)b.src[t] + at * (dt == F32 ? 4 : 2);
        int done = 0;
        if ((uintptr_t)p % 16 == 0) {
            const u32x4* q = (const u32x4*)p;
            if (dt == F32) {
                const int n4 = n / 4;
                for (int i = threadIdx.x; i < n4; i += 256) {
                    const u32x4 u = q[i];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)
                        add<KIND>(acc[j], __uint_as_float(u[j]));
                }
                done = n4 * 4;
            } else {
                const int n8 = n / 8;
                for (int i = threadIdx.x; i < n8; i += 256) {
                    const u32x4 u = q[i];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        add<KIND>(acc[j], lo16(u[j], dt));
                        add<KIND>(acc[j], hi16(u[j], dt));
                    }
                }
                done = n8 * 8;
            }
        }
        for (int i = done + threadIdx.x; i < n; i += 256)
            add<KIND>(acc[0], load1(p, i, dt));
    }
    const double v = block_total<KIND>(both<KIND>(both<KIND>(acc[0], acc[1]),
                                                  both<KIND>(acc[2], acc[3])));
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

template <int KIND>
__global__ __launch_bounds__(256)
void finish_kernel(const double* __restrict__ part, int n, double max_norm,
                   float* __restrict__ norm, double* __restrict__ factor) {
    double v = 0;
    for (int i = threadIdx.x; i < n; i += 256) v = both<KIND>(v, part[i]);
    v = block_total<KIND>(v);
    if (threadIdx.x) return;
    if (KIND == L2) v = __builtin_sqrt(v);
    norm[0] = (float)v;
    const double f = max_norm / (v + 1e-6);
    factor[0] = f > 1.0 ? 1.0 : f;       // a NaN stays
}

__global__ __launch_bounds__(256)
void scale_kernel(const Batch b, const double* __restrict__ factor) {
    const double f = factor[0];
    const float f32 = (float)f;
    const int chunks = b.first[b.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = tensor_of(b, c);
        const int sd = b.src_dt[t], dd = b.dst_dt[t];
        // nothing to scale, nothing to move
        if (f == 1.0 && b.src[t] == b.dst[t]) continue;
        const int64_t at = (int64_t)(c - b.first[t]) * CHUNK;
        const int n = (int)min((int64_t)CHUNK, b.n[t] - at);
        const char* p = (const char*)b.src[t] + at * (sd == F32 ? 4 : 2);
        char* q = (char*)b.dst[t] + at * (dd == F32 ? 4 : 2);
        int done = 0;
        if (sd == dd && ((uintptr_t)p | (uintptr_t)q) % 16 == 0) {
            const u32x4* pu = (const u32x4*)p;
            u32x4* qu = (u32x4*)q;
            if (sd == F32) {
                const int n4 = n / 4;
                for (int i = threadIdx.x; i < n4; i += 256) {
                    u32x4 u = pu[i];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j)    // one rounding, from 64 bits
                        u[j] = __float_as_uint(
                            (float)((double)__uint_as_float(u[j]) * f));
                    qu[i] = u;
                }
                done = n4 * 4;
            } else {
                const int n8 = n / 8;
                for (int i = threadIdx.x; i < n8; i += 256) {
                    u32x4 u = pu[i];
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float a = lo16(u[j], sd) * f32;
                        const float h = hi16(u[j], sd) * f32;
                        unsigned short x, y;
                        if (sd == BF16) {
                            x = __builtin_bit_cast(unsigned short, (__bf16)a);
                            y = __builtin_bit_cast(unsigned short, (__bf16)h);
                        } else {
                            x = __builtin_bit_cast(unsigned short, (_Float16)a);
                            y = __builtin_bit_cast(unsigned short, (_Float16)h);
                        }
                        u[j] = x | (unsigned)y << 16;
                    }
                    qu[i] = u;
                }
                done = n8 * 8;
            }
        }
        for (int i = done + threadIdx.x; i < n; i += 256)
            store1(q, i, dd, (float)((double)load1(p, i, sd) * f));
    }
}

// the list in batches; empty tensors are left out
template <class F>
void for_batches(const std::vector<Item>& items, F&& f) {
    Batch b;
    b.count = 0;
    int chunks = 0;
    auto flush = [&]() {
        if (!b.count) return;
        b.first[b.count] = chunks;
        f(b, chunks < BLOCKS ? chunks : BLOCKS);
        b.count = 0;
        chunks = 0;
    };
    for (const Item& it : items) {
        if (!it.n) continue;
        const int64_t c = (it.n + CHUNK - 1) / CHUNK;
        if (b.count == TENSORS || chunks + c > INT32_MAX) flush();
        b.src[b.count] = it.src;
        b.dst[b.count] = it.dst;
        b.n[b.count] = it.n;
        b.first[b.count] = chunks;
        b.src_dt[b.count] = (uint8_t)it.src_dt;
        b.dst_dt[b.count] = (uint8_t)it.dst_dt;
        ++b.count;
        chunks += (int)c;
    }
    flush();
}

}  // namespace

size_t workspace_doubles(const std::vector<Item>& items) {
    size_t n = 1;
    for_batches(items, [&](const Batch&, int blocks) { n += blocks; });
    return n;
}

void norm(const std::vector<Item>& items, int kind, double max_norm,
          float* norm, double* work, hipStream_t stream) {
    int n = 0;
    #define GC_KIND(CALL) \
        do { if (kind == L2) { CALL(L2); } \
             else if (kind == L1) { CALL(L1); } \
             else { CALL(LINF); } } while (0)
    for_batches(items, [&](const Batch& b, int blocks) {
        #define GC_N(K) hipLaunchKernelGGL((norm_kernel<K>), dim3(blocks), \
                                           dim3(256), 0, stream, b, work + 1 + n)
        GC_KIND(GC_N);
        #undef GC_N
        n += blocks;
    });
    #define GC_F(K) hipLaunchKernelGGL((finish_kernel<K>), dim3(1), dim3(256), \
                                       0, stream, work + 1, n, max_norm, norm, work)
    GC_KIND(GC_F);
    #undef GC_F
    #undef GC_KIND
}

void scale(const std::vector<Item>& items, const double* work,
           hipStream_t stream) {
    for_batches(items, [&](const Batch& b, int blocks) {
        hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(256), 0, stream, b,
                           work);
    });
}

}  // namespace gradclip
