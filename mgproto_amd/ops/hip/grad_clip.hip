// Global gradient norm and clipping over many tensors.
//
//   N = (sum_t sum_i |g|^p)^(1/p), p = 1, 2 or infinity
//   g <- g * min(1, max_norm / (N + 1e-6))
//
// Bound by memory: the list is read for the norm, then read and written once
// to be scaled. Sums are held in 64 bits: squares of large fp32 values leave the range of
// fp32, and at one 64-bit multiply-add an element the vector units are far from
// their limit.
//
// The list travels in the kernels' own arguments, up to MANY tensors a launch: nothing is uploaded, so a captured graph holds everything it needs
// and a call never waits for the host. All loads of a chunk are sent before the
// first is used. Every sum has a fixed order, and each block of the second pass
// adds up the blocks' sums itself, which saves a launch: five small tensors take
// 9.4 us, bound by the host.
//
// 1.34e9 bf16 elements in 64 tensors: norm 452 us (5.9 TB/s), all 1514; a copy of
// 1 GiB runs at 5.1 TB/s. Blocks of the first pass take runs of chunks (every
// 1024th chunk: 470); those of the second, which writes as well, every 2048th
// (runs: 1545), and past the caches (120 Mi fp32 elements in 60 odd tensors: 254
// against 281).

#include <hip/hip_runtime.h>

#include "grad_clip.h"

namespace gradclip {
namespace {

constexpr int F32 = 0, BF16 = 1;         // 2 = fp16
constexpr int FEW = 16, MANY = 180;      // tensors of a launch: 400 bytes, or 4 KB
constexpr int LOADS = 4;                 // of 16 bytes a thread and chunk
constexpr int CHUNK = 256 * LOADS * 16;  // bytes of the source
constexpr int NORM_BLOCKS = 1024;        // of a launch, at most
constexpr int SCALE_BLOCKS = 2048;
constexpr int PARTS = 2 * NORM_BLOCKS;   // sums that a block adds up by itself

template <int TENSORS>
struct Batch {
    const void* src[TENSORS];
    void* dst[TENSORS];
    // first chunk (28 bits), and above them type of src + 3 * type of dst
    unsigned first[TENSORS + 1];
    uint16_t last[TENSORS];              // elements of the last chunk, less 1
    int count;
};
static_assert(sizeof(Batch<MANY>) <= 4000, "kernel arguments");

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

static __host__ __device__ constexpr int elements(int dt) {   // of a chunk
    return CHUNK / (dt == F32 ? 4 : 2);
}

template <int DT> struct Type { typedef float T; };
template <> struct Type<BF16> { typedef __bf16 T; };
template <> struct Type<2> { typedef _Float16 T; };

// E consecutive elements anywhere, moved 16 bytes at a time where they fill them
template <int DT, int E>
union Unit {
    typedef typename Type<DT>::T T;
    static constexpr int B = E * sizeof(T) < 16 ? 8 : 16;
    typedef unsigned Word __attribute__((ext_vector_type(B / 4)));
    struct __attribute__((packed, aligned(sizeof(T)))) Any { Word u; };
    T v[E];
    Word u[E * sizeof(T) / B];
    __device__ __forceinline__ void load(const void* p) {
        #pragma unroll
        for (int i = 0; i < (int)(E * sizeof(T)) / B; ++i)
            u[i] = reinterpret_cast<const Any*>(p)[i].u;
    }
    __device__ __forceinline__ void store(void* p) const {
        typedef Word Loose __attribute__((aligned(sizeof(T))));
        #pragma unroll
        for (int i = 0; i < (int)(E * sizeof(T)) / B; ++i)
            __builtin_nontemporal_store(u[i], reinterpret_cast<Loose*>(p) + i);
    }
};

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

template <int T>
static __host__ __device__ __forceinline__ int chunk_of(const Batch<T>& b, int t) {
    return (int)(b.first[t] & 0x0fffffffu);
}

// Some of the chunks, in their order, with their tensors.
template <int T>
struct Walk {
    int c, end, inc, t, from, next;      // next: the next tensor's first chunk
    __device__ __forceinline__ Walk(const Batch<T>& b, int c, int end, int inc)
        : c(c), end(end), inc(inc) {
        int lo = 0, hi = b.count - 1;    // the last with first <= c
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (chunk_of(b, mid) <= c) lo = mid; else hi = mid - 1;
        }
        t = lo, from = chunk_of(b, t), next = chunk_of(b, t + 1);
    }
    __device__ __forceinline__ bool done() const { return c >= end; }
    __device__ __forceinline__ void step(const Batch<T>& b) {
        c += inc;
        if (c < end)
            while (c >= next) from = next, next = chunk_of(b, ++t + 1);
    }
    __device__ __forceinline__ int types(const Batch<T>& b) const {
        return (int)(b.first[t] >> 28);
    }
    __device__ __forceinline__ int length(const Batch<T>& b, int dt) const {
        return c + 1 == next ? b.last[t] + 1 : elements(dt);
    }
};

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

template <int KIND, int DT>
static __device__ __forceinline__ void add_chunk(double (&acc)[4],
                                                 const void* src, int64_t at,
                                                 int n) {
    typedef typename Type<DT>::T T;
    constexpr int E = 16 / sizeof(T);
    const T* p = reinterpret_cast<const T*>(src) + at;
    if (n == elements(DT)) {
        Unit<DT, E> u[LOADS];
        #pragma unroll
        for (int i = 0; i < LOADS; ++i) u[i].load(p + (i * 256 + threadIdx.x) * E);
        #pragma unroll
        for (int i = 0; i < LOADS; ++i)
            #pragma unroll
            for (int e = 0; e < E; ++e) add<KIND>(acc[e & 3], (float)u[i].v[e]);
        return;
    }
    const int whole = n / E;
    for (int i = threadIdx.x; i < whole; i += 256) {
        Unit<DT, E> u;
        u.load(p + i * E);
        #pragma unroll
        for (int e = 0; e < E; ++e) add<KIND>(acc[e & 3], (float)u.v[e]);
    }
    const int i = whole * E + threadIdx.x;
    if (i < n) add<KIND>(acc[0], (float)p[i]);
}

template <int KIND, int T>
__global__ __launch_bounds__(256)
void norm_kernel(const Batch<T> b, double* __restrict__ part) {
    double acc[4] = {0, 0, 0, 0};
    const long chunks = chunk_of(b, b.count);
    const int lo = (int)(chunks * blockIdx.x / gridDim.x);
    const int hi = (int)(chunks * (blockIdx.x + 1) / gridDim.x);
    for (Walk<T> r(b, lo, hi, 1); !r.done(); r.step(b)) {
        const int dt = r.types(b) % 3;
        const int n = r.length(b, dt);
        const int64_t at = (int64_t)(r.c - r.from) * elements(dt);
        if (dt == F32) add_chunk<KIND, F32>(acc, b.src[r.t], at, n);
        else if (dt == BF16) add_chunk<KIND, BF16>(acc, b.src[r.t], at, n);
        else add_chunk<KIND, 2>(acc, b.src[r.t], at, n);
    }
    const double v = block_total<KIND>(both<KIND>(both<KIND>(acc[0], acc[1]),
                                                  both<KIND>(acc[2], acc[3])));
    if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// the sum (or maximum) of n sums, in every thread of a block
template <int KIND>
static __device__ __forceinline__ double add_parts(const double* part, int n) {
    double v = 0;
    #pragma unroll 4
    for (int i = threadIdx.x; i < n; i += 256) v = both<KIND>(v, part[i]);
    return block_total<KIND>(v);
}
template <int KIND>
static __device__ __forceinline__ double root(double v) {
    return KIND == L2 ? __builtin_sqrt(v) : v;
}

// sum[0] = the sum of n sums, norm[0] = the norm
template <int KIND>
__global__ __launch_bounds__(256)
void finish_kernel(const double* __restrict__ part, int n,
                   double* __restrict__ sum, float* __restrict__ norm) {
    const double v = add_parts<KIND>(part, n);
    if (threadIdx.x) return;
    sum[0] = v;
    norm[0] = (float)root<KIND>(v);
}

// 64 bits where either type has 32, rounded once: on the way to 16 bits the 32 in
// between are rounded to odd (by truncation, the last bit set where something was
// lost), which keeps an element next to the middle of two values on its side. From 16
// bits to 16, the factor f = m 2^e is rounded to 32 (m, between 1/2 and 1) and so is
// the product: two times 2^-24 beside the result's 2^-9 or 2^-12. Its exponent comes
// last: the norm of bf16 gradients may pass 2^128, and the factor then lies below
// what 32 bits hold, where the products need not.
template <int SD, int DD>
static __device__ __forceinline__ typename Type<DD>::T scaled(
        typename Type<SD>::T v, double f, float m, int e) {
    if constexpr (SD == F32 || DD == F32) {
        const double d = (double)(float)v * f;
        float r = (float)d;
        if constexpr (DD != F32) {
            if ((double)r != d) {
                unsigned b = __float_as_uint(r);
                b -= __builtin_fabs((double)r) > __builtin_fabs(d);
                r = __uint_as_float(b | 1u);
            }
        }
        return (typename Type<DD>::T)r;
    } else return (typename Type<DD>::T)__builtin_ldexpf((float)v * m, e);
}

template <int SD, int DD>
static __device__ __forceinline__ void scale_chunk(const void* src, void* dst,
                                                   int64_t at, int n, double f) {
    typedef typename Type<SD>::T S;
    typedef typename Type<DD>::T D;
    constexpr int E = 16 / sizeof(S);
    const S* p = reinterpret_cast<const S*>(src) + at;
    D* q = reinterpret_cast<D*>(dst) + at;
    int e = 0;
    const float m = (float)frexp(f, &e);
    if (n == elements(SD)) {
        Unit<SD, E> u[LOADS];
        #pragma unroll
        for (int i = 0; i < LOADS; ++i) u[i].load(p + (i * 256 + threadIdx.x) * E);
        #pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            Unit<DD, E> o;
            #pragma unroll
            for (int j = 0; j < E; ++j) o.v[j] = scaled<SD, DD>(u[i].v[j], f, m, e);
            o.store(q + (i * 256 + threadIdx.x) * E);
        }
        return;
    }
    const int whole = n / E;
    for (int i = threadIdx.x; i < whole; i += 256) {
        Unit<SD, E> u;
        Unit<DD, E> o;
        u.load(p + i * E);
        #pragma unroll
        for (int j = 0; j < E; ++j) o.v[j] = scaled<SD, DD>(u.v[j], f, m, e);
        o.store(q + i * E);
    }
    const int i = whole * E + threadIdx.x;
    if (i < n) q[i] = scaled<SD, DD>(p[i], f, m, e);
}

template <int KIND, int T>
__global__ __launch_bounds__(256)
void scale_kernel(const Batch<T> b, const double* __restrict__ part, int n_parts,
                  double max_norm, float* __restrict__ norm) {
    const double v = root<KIND>(add_parts<KIND>(part, n_parts));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)v;
    double f = max_norm / (v + 1e-6);
    f = f > 1.0 ? 1.0 : f;               // a NaN stays
    for (Walk<T> r(b, blockIdx.x, chunk_of(b, b.count), gridDim.x); !r.done();
         r.step(b)) {
        const void* src = b.src[r.t];
        void* dst = b.dst[r.t];
        // nothing to scale, nothing to move
        if (f == 1.0 && src == dst) continue;
        const int types = r.types(b), sd = types % 3;
        const int n = r.length(b, sd);
        const int64_t at = (int64_t)(r.c - r.from) * elements(sd);
        switch (types) {
            case 0: scale_chunk<0, 0>(src, dst, at, n, f); break;
            case 1: scale_chunk<1, 0>(src, dst, at, n, f); break;
            case 2: scale_chunk<2, 0>(src, dst, at, n, f); break;
            case 3: scale_chunk<0, 1>(src, dst, at, n, f); break;
            case 4: scale_chunk<1, 1>(src, dst, at, n, f); break;
            case 5: scale_chunk<2, 1>(src, dst, at, n, f); break;
            case 6: scale_chunk<0, 2>(src, dst, at, n, f); break;
            case 7: scale_chunk<1, 2>(src, dst, at, n, f); break;
            default: scale_chunk<2, 2>(src, dst, at, n, f); break;
        }
    }
}

constexpr int64_t CHUNKS = 1L << 28;     // of a launch, fewer than that

int64_t chunks_of(const Item& it) {
    return (it.n + elements(it.src_dt) - 1) / elements(it.src_dt);
}

// The list in batches; empty tensors are left out.
template <int T>
std::vector<Batch<T>> batches(const std::vector<Item>& items) {
    std::vector<Batch<T>> list;
    int64_t chunks = CHUNKS;
    for (const Item& it : items) {
        if (!it.n) continue;
        const int64_t c = chunks_of(it);
        if (list.empty() || list.back().count == T || chunks + c >= CHUNKS) {
            list.emplace_back();
            list.back().count = 0;
            chunks = 0;
        }
        Batch<T>& b = list.back();
        const int t = b.count++;
        b.src[t] = it.src;
        b.dst[t] = it.dst;
        b.first[t] = (unsigned)chunks
            | (unsigned)(it.src_dt + 3 * it.dst_dt) << 28;
        b.last[t] = (uint16_t)(it.n - (c - 1) * elements(it.src_dt) - 1);
        chunks += c;
        b.first[t + 1] = (unsigned)chunks;
    }
    return list;
}

template <int T>
int blocks_of(const Batch<T>& b, int most) {
    const int chunks = chunk_of(b, b.count);
    return chunks < most ? chunks : most;
}

}  // namespace

struct List::Data {
    std::vector<Batch<FEW>> few;         // one of the two is empty
    std::vector<Batch<MANY>> many;
    template <class F> void each(F&& f) const {
        for (const auto& b : few) f(b);
        for (const auto& b : many) f(b);
    }
};

// Few tensors: the arguments are read from the host's memory, and ten times
// fewer of them take a list of five from 10.9 to 9.4 us.
List::List(const std::vector<Item>& items) : d(new Data) {
    if (items.size() <= FEW) d->few = batches<FEW>(items);
    else d->many = batches<MANY>(items);
}
List::~List() { delete d; }

size_t List::workspace_doubles() const {
    return 1 + (d->few.size() + d->many.size()) * NORM_BLOCKS;
}

#define GC_KIND(CALL) do { if (kind == L2) { CALL(L2); } \
                           else if (kind == L1) { CALL(L1); } \
                           else { CALL(LINF); } } while (0)

template <int T>
static void launch_norm(const Batch<T>& b, int kind, int blocks, double* part,
                        hipStream_t stream) {
    #define GC_N(K) hipLaunchKernelGGL((norm_kernel<K, T>), dim3(blocks), \
                                       dim3(256), 0, stream, b, part)
    GC_KIND(GC_N);
    #undef GC_N
}
template <int T>
static void launch_scale(const Batch<T>& b, int kind, const double* part, int n,
                         double max_norm, float* norm, hipStream_t stream) {
    #define GC_S(K) hipLaunchKernelGGL((scale_kernel<K, T>), \
        dim3(blocks_of(b, SCALE_BLOCKS)), dim3(256), 0, stream, b, part, n, \
        max_norm, norm)
    GC_KIND(GC_S);
    #undef GC_S
}

int List::sums(int kind, double* part, hipStream_t stream) const {
    int n = 0;
    d->each([&](const auto& b) {
        const int blocks = blocks_of(b, NORM_BLOCKS);
        launch_norm(b, kind, blocks, part + n, stream);
        n += blocks;
    });
    return n;
}

static void finish(int kind, const double* part, int n, double* sum, float* norm,
                   hipStream_t stream) {
    #define GC_F(K) hipLaunchKernelGGL((finish_kernel<K>), dim3(1), dim3(256), \
                                       0, stream, part, n, sum, norm)
    GC_KIND(GC_F);
    #undef GC_F
}

void List::norm(int kind, float* norm, double* work, hipStream_t stream) const {
    const int n = sums(kind, work + 1, stream);
    finish(kind, work + 1, n, work, norm, stream);
}

void List::clip(int kind, double max_norm, float* norm, double* work,
                hipStream_t stream) const {
    const double* part = work + 1;
    int n = sums(kind, work + 1, stream);
    if (n == 0 || n > PARTS) {           // nothing to scale, or long lists
        finish(kind, part, n, work, norm, stream);
        part = work, n = 1, norm = nullptr;
    }
    d->each([&](const auto& b) {
        launch_scale(b, kind, part, n, max_norm, norm, stream);
        norm = nullptr;
    });
}

}  // namespace gradclip
