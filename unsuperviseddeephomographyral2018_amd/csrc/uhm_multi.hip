// uhm_multi.hip -- global gradient norm over many tensors, clipping by it, and the Adam update that clips on the way (gfx950).
//
//   n = sqrt(sum_i sum_j t_ij^2)        f = n > clip ? clip / n : 1   (NaN when n is not finite)
//   clip: out = f t                     adam: g = f grad; m, v, p as in the header
//
// All three stream their tensors and compute next to nothing: what bounds them is HBM bandwidth for the regressor's 34 M
// elements and launch latency for lists of small tensors.  So a list of any composition takes TWO launches, not one per tensor
// (a few more past a table's 256, 128 or 64 tensors):
//   1  sum_squares : block b adds the squares of its chunks in f64 and stores one partial sum;
//   2  scale / adam: every block adds ALL partial sums again (a few thousand doubles out of the L2, in a fixed order, while its
//      first tensor loads are in flight) -- no third launch to finish the norm, no ticket that a replay would have to reset.
// The tensors' addresses travel in the kernel's arguments (a table of up to TENSORS entries per launch), so nothing is copied to
// the device first and a captured graph holds them.  A chunk is CHUNK elements of ONE tensor; block b takes chunks b, b + grid,
// b + 2 grid, ... of the concatenated chunk list, a fixed assignment, so that sums do not depend on timing.
// f64 sums: squares of f32 neither overflow (|t| up to 3e38) nor vanish (down to 1e-45), and the kernel stays memory-bound
// (one f64 FMA per element at half the f32 rate).
// One MI355X, us a pass: norm of the 128 px regressor's gradients (137 MB) 28.5, of 300 small tensors 18; clipping 70.7 / 40 small ones
// 18; Adam with clipping 182 (957 MB without the second read of the gradients: 5.3 TB/s), at 32 px (77 MB) 19.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>
#include "../../include/uh_model_ops.h"

namespace uhm {

constexpr int THREADS = 256;
constexpr int CHUNK = 4096;              // elements
constexpr int MAX_GRID = 2048;           // 256 CUs x 8 blocks of 4 waves
constexpr unsigned NO_CHUNK = 0xffffffffu;

// The table of one launch: 8 bytes a pointer and 6 more per tensor, so that long lists take few launches (each costs the host 2.5 us).
// first[i]: index of tensor i's first chunk; entries past the last tensor hold NO_CHUNK.  info[i]: type, alignment, and by how much
// the tensor ends before its last chunk does.
constexpr unsigned TYPE_BITS = 3, ALIGNED_BIT = 4, SHORT_SHIFT = 3;
static_assert((CHUNK - 1) << SHORT_SHIFT <= 0xffff, "info has 16 bits");
template <int POINTERS, int TENSORS>
struct Table {
    void* p[POINTERS][TENSORS];
    unsigned first[TENSORS];
    unsigned short info[TENSORS];
    unsigned chunks;
};
// (the argument segment of a kernel is kept below 4 KB)
using NormTable = Table<1, 256>;
using ClipTable = Table<2, 128>;
using AdamTable = Table<4, 64>;
static_assert(sizeof(NormTable) < 4000 && sizeof(ClipTable) < 4000 && sizeof(AdamTable) < 4000, "kernel arguments");

// one chunk of a table: which tensor, which of its elements
struct Part { int tensor, type; bool aligned; long long begin, end; };

// the tensor that holds chunk c: how many first[] are <= c, less one.  One ballot per 64 entries.
template <int POINTERS, int N>
__device__ __forceinline__ Part find(const Table<POINTERS, N>& t, unsigned c) {
    const int lane = threadIdx.x & 63;
    int i = -1;
#pragma unroll
    for (int k = 0; k < N; k += 64) i += __popcll(__ballot(t.first[k + lane] <= c));
    i = __builtin_amdgcn_readfirstlane(i);
    const unsigned next = i + 1 < N ? min(t.first[i + 1 < N ? i + 1 : i], t.chunks) : t.chunks, info = t.info[i];
    Part p = {i, (int)(info & TYPE_BITS), (info & ALIGNED_BIT) != 0, (long long)(c - t.first[i]) * CHUNK, 0};
    p.end = p.begin + CHUNK - (c + 1 == next ? info >> SHORT_SHIFT : 0);
    return p;
}

// 16 bytes to or from memory past the caches, for lists that they cannot hold anyway
typedef unsigned u4 __attribute__((ext_vector_type(4)));
template <bool STREAM, typename T>
__device__ __forceinline__ T fetch(const T* p) {
    static_assert(sizeof(T) == 16, "16 bytes");
    if constexpr (STREAM) return __builtin_bit_cast(T, __builtin_nontemporal_load(reinterpret_cast<const u4*>(p)));
    else return *p;
}
template <bool STREAM, typename T>
__device__ __forceinline__ void store(T* p, const T& v) {
    if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(u4, v), reinterpret_cast<u4*>(p));
    else *p = v;
}

__device__ __forceinline__ float from_bf16(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
__device__ __forceinline__ float from_f16(unsigned short b) { return __half2float(__ushort_as_half(b)); }
__device__ __forceinline__ unsigned short to_bf16(float f) { return __builtin_bit_cast(unsigned short, (__bf16)f); }  // nearest even
__device__ __forceinline__ unsigned short to_f16(float f) { return __half_as_ushort(__float2half(f)); }               // nearest even

template <int T> struct Type;
template <> struct Type<UHM_F32> {
    using raw = float;
    static __device__ __forceinline__ float get(raw r) { return r; }
    static __device__ __forceinline__ raw put(float f) { return f; }
};
template <> struct Type<UHM_BF16> {
    using raw = unsigned short;
    static __device__ __forceinline__ float get(raw r) { return from_bf16(r); }
    static __device__ __forceinline__ raw put(float f) { return to_bf16(f); }
};
template <> struct Type<UHM_F16> {
    using raw = unsigned short;
    static __device__ __forceinline__ float get(raw r) { return from_f16(r); }
    static __device__ __forceinline__ raw put(float f) { return to_f16(f); }
};

// 16 bytes of a tensor: 4 f32 or 8 16-bit elements
template <int T>
struct alignas(16) Vec {
    static constexpr int N = 16 / sizeof(typename Type<T>::raw);
    typename Type<T>::raw v[N];
};

// f(lowest .. ) over the elements [begin, end) of this block's chunk: `vec(i)` on full 16-byte vectors, `one(i)` on the rest
template <int N, typename V, typename O>
__device__ __forceinline__ void over_chunk(long long begin, long long end, bool aligned, V vec, O one) {
    if (aligned) {
        if (end - begin == CHUNK) {
#pragma unroll
            for (int k = 0; k < CHUNK / (THREADS * N); ++k) vec(begin + (long long)(k * THREADS + threadIdx.x) * N);
            return;
        }
        const long long whole = begin + (end - begin) / N * N;
        for (long long i = begin + (long long)threadIdx.x * N; i < whole; i += THREADS * N) vec(i);
        begin = whole;
    }
    for (long long i = begin + threadIdx.x; i < end; i += THREADS) one(i);
}

__device__ __forceinline__ double block_sum(double s) {
    __shared__ double sm[THREADS / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) s += __shfl_down(s, d, 64);
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) s += sm[w];
    return s;                            // the same in every thread
}

template <int T>
__device__ __forceinline__ double squares(const void* p, long long begin, long long end, bool aligned) {
    const auto* q = (const typename Type<T>::raw*)p;
    double s0 = 0.0, s1 = 0.0;
    over_chunk<Vec<T>::N>(begin, end, aligned,
        [&](long long i) {
            const Vec<T> x = *reinterpret_cast<const Vec<T>*>(q + i);
#pragma unroll
            for (int e = 0; e < Vec<T>::N; e += 2) {
                const double a = Type<T>::get(x.v[e]), b = Type<T>::get(x.v[e + 1]);
                s0 = fma(a, a, s0);
                s1 = fma(b, b, s1);
            }
        },
        [&](long long i) { const double a = Type<T>::get(q[i]); s0 = fma(a, a, s0); });
    return s0 + s1;
}

__global__ __launch_bounds__(THREADS) void sum_squares_kernel(const NormTable t, double* __restrict__ partial) {
    double s = 0.0;
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Part h = find(t, c);
        const void* p = t.p[0][h.tensor];
        switch (h.type) {
            case UHM_F32: s += squares<UHM_F32>(p, h.begin, h.end, h.aligned); break;
            case UHM_BF16: s += squares<UHM_BF16>(p, h.begin, h.end, h.aligned); break;
            default: s += squares<UHM_F16>(p, h.begin, h.end, h.aligned); break;
        }
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// the norm from the partial sums: every thread adds partial[tid], partial[tid + 256], ... in order, then the block
__device__ __forceinline__ float norm_of(const double* __restrict__ partial, int count) {
    double s = 0.0;
    for (int k = threadIdx.x; k < count; k += THREADS) s += partial[k];
    return (float)sqrt(block_sum(s));
}

__global__ __launch_bounds__(THREADS) void finish_norm_kernel(const double* __restrict__ partial, int count, float* __restrict__ norm) {
    const float n = norm_of(partial, count);
    if (threadIdx.x == 0) norm[0] = n;
}

// f as a product first * rest.  A quotient below 2^-126 would keep few of its bits in f32 (3e38 clipped to 1e-3: 2e-4 off): it is kept 2^126
// times as large (clip < 4 there, so that nothing overflows) and rest, otherwise 1, takes that back, exactly.
struct Factor {
    float first, rest;
    __device__ __forceinline__ float operator()(float x) const { return x * first * rest; }
    __device__ __forceinline__ bool changes_nothing() const { return first == 1.0f && rest == 1.0f; }
};
__device__ __forceinline__ Factor clip_factor(float n, float clip) {
    if (!(n < INFINITY)) return {__builtin_nanf(""), 1.0f};      // inf or NaN (a norm is never negative)
    if (!(n > clip)) return {1.0f, 1.0f};
    const float f = clip / n;
    if (f >= 0x1p-126f) return {f, 1.0f};
    return {clip * 0x1p126f / n, 0x1p-126f};
}

template <int T, bool STREAM>
__device__ __forceinline__ void scale(const void* p, void* out, const Factor f, long long begin, long long end, bool aligned) {
    const auto* q = (const typename Type<T>::raw*)p;
    auto* o = (typename Type<T>::raw*)out;
    over_chunk<Vec<T>::N>(begin, end, aligned,
        [&](long long i) {
            Vec<T> x = *reinterpret_cast<const Vec<T>*>(q + i);
#pragma unroll
            for (int e = 0; e < Vec<T>::N; ++e) x.v[e] = Type<T>::put(f(Type<T>::get(x.v[e])));   // one rounding to the type
            store<STREAM>(reinterpret_cast<Vec<T>*>(o + i), x);
        },
        [&](long long i) { o[i] = Type<T>::put(f(Type<T>::get(q[i]))); });
}

// The order of a table's chunks in the second pass.  STREAM: lists that the caches do not hold.  The last tensors that the first
// pass read may still be there, so it goes backwards, and what it alone touches goes past the caches (loads and stores marked as
// not to be kept), which leaves the gradients their place.  Regressor at 128 px (34 M elements): clipping 87.1 -> 73.3 us,
// Adam 215.5 -> 183.1 us; at 32 px (2.7 M), whose 77 MB the 256 MB cache holds from step to step, Adam 20.6 us without and 23.6 with.
template <bool STREAM>
__device__ __forceinline__ unsigned in_order(unsigned c, unsigned chunks) { return STREAM ? chunks - 1 - c : c; }

template <bool STREAM>
__global__ __launch_bounds__(THREADS) void scale_kernel(const ClipTable t, const double* __restrict__ partial, int count,
                                                        const float* __restrict__ use_norm, float clip, float* __restrict__ norm) {
    const float n = use_norm ? use_norm[0] : norm_of(partial, count);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = n;
    const Factor f = clip_factor(n, clip);
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Part h = find(t, in_order<STREAM>(c, t.chunks));
        const void* p = t.p[0][h.tensor];
        void* o = t.p[1][h.tensor];
        if (p == o && f.changes_nothing()) continue;               // in place and nothing to clip: the values are there
        switch (h.type) {
            case UHM_F32: scale<UHM_F32, STREAM>(p, o, f, h.begin, h.end, h.aligned); break;
            case UHM_BF16: scale<UHM_BF16, STREAM>(p, o, f, h.begin, h.end, h.aligned); break;
            default: scale<UHM_F16, STREAM>(p, o, f, h.begin, h.end, h.aligned); break;
        }
    }
}

struct AdamScalars { float beta1, one_minus_beta1, beta2, one_minus_beta2, step_size, inv_sqrt_bias2, eps; };

__device__ __forceinline__ void adam_one(float& p, float g, float& m, float& v, const AdamScalars& a) {
    m = a.beta1 * m + a.one_minus_beta1 * g;
    v = a.beta2 * v + a.one_minus_beta2 * (g * g);
    p = p - a.step_size * (m / (sqrtf(v) * a.inv_sqrt_bias2 + a.eps));
}

template <int T, bool STREAM>
__device__ __forceinline__ void adam(float* p, const void* grad, float* m, float* v, const Factor f, const AdamScalars& a, long long begin,
                                     long long end, bool aligned) {
    const auto* g = (const typename Type<T>::raw*)grad;
    struct alignas(sizeof(typename Type<T>::raw) * 4) G4 { typename Type<T>::raw v[4]; };
    over_chunk<4>(begin, end, aligned,
        [&](long long i) {
            float4 pp = fetch<STREAM>(reinterpret_cast<const float4*>(p + i)), mm = fetch<STREAM>(reinterpret_cast<const float4*>(m + i)),
                   vv = fetch<STREAM>(reinterpret_cast<const float4*>(v + i));
            const G4 gg = *reinterpret_cast<const G4*>(g + i);
            adam_one(pp.x, f(Type<T>::get(gg.v[0])), mm.x, vv.x, a);
            adam_one(pp.y, f(Type<T>::get(gg.v[1])), mm.y, vv.y, a);
            adam_one(pp.z, f(Type<T>::get(gg.v[2])), mm.z, vv.z, a);
            adam_one(pp.w, f(Type<T>::get(gg.v[3])), mm.w, vv.w, a);
            store<STREAM>(reinterpret_cast<float4*>(p + i), pp);
            store<STREAM>(reinterpret_cast<float4*>(m + i), mm);
            store<STREAM>(reinterpret_cast<float4*>(v + i), vv);
        },
        [&](long long i) { adam_one(p[i], f(Type<T>::get(g[i])), m[i], v[i], a); });
}

template <bool STREAM>
__global__ __launch_bounds__(THREADS) void adam_kernel(const AdamTable t, const double* __restrict__ partial, int count,
                                                       const float* __restrict__ use_norm, float clip, int skip_nonfinite,
                                                       const AdamScalars a, float* __restrict__ norm) {
    const float n = use_norm ? use_norm[0] : norm_of(partial, count);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = n;
    if (skip_nonfinite && !(n < INFINITY)) return;
    const Factor f = clip_factor(n, clip);
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Part h = find(t, in_order<STREAM>(c, t.chunks));
        const int i = h.tensor;
        float *p = (float*)t.p[0][i], *m = (float*)t.p[2][i], *v = (float*)t.p[3][i];
        switch (h.type) {
            case UHM_F32: adam<UHM_F32, STREAM>(p, t.p[1][i], m, v, f, a, h.begin, h.end, h.aligned); break;
            case UHM_BF16: adam<UHM_BF16, STREAM>(p, t.p[1][i], m, v, f, a, h.begin, h.end, h.aligned); break;
            default: adam<UHM_F16, STREAM>(p, t.p[1][i], m, v, f, a, h.begin, h.end, h.aligned); break;
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
inline long long chunks_of(long long n) { return (n + CHUNK - 1) / CHUNK; }
inline size_t elem_size(int dtype) { return dtype == UHM_F32 ? 4 : 2; }

// walks a list in tables of up to TENSORS non-empty tensors: `launch(table, grid)` for each
template <typename TABLE, int POINTERS, int TENSORS, typename F>
int for_tables(const void* const* const (&lists)[POINTERS], const long long* numel, const int* dtypes, int count, F launch) {
    TABLE t{};
    int k = 0;
    long long chunks = 0;
    auto flush = [&]() -> int {
        if (k == 0) return 0;
        for (int j = k; j < TENSORS; ++j) t.first[j] = NO_CHUNK;
        t.chunks = (unsigned)chunks;
        const unsigned grid = (unsigned)(chunks < MAX_GRID ? chunks : MAX_GRID);
        k = 0;
        chunks = 0;
        return launch(t, grid);
    };
    for (int i = 0; i < count; ++i) {
        if (numel[i] == 0) continue;
        uintptr_t bits = 0;
        for (int j = 0; j < POINTERS; ++j) {
            t.p[j][k] = const_cast<void*>(lists[j][i]);
            bits |= (uintptr_t)lists[j][i];
        }
        t.first[k] = (unsigned)chunks;
        chunks += chunks_of(numel[i]);
        t.info[k] = (unsigned short)((unsigned)dtypes[i] | ((bits & 15) == 0 ? ALIGNED_BIT : 0) |
                                     (unsigned)(chunks_of(numel[i]) * CHUNK - numel[i]) << SHORT_SHIFT);
        if (++k == TENSORS)
            if (int e = flush()) return e;
    }
    return flush();
}

int check_list(const void* const* tensors, const long long* numel, const int* dtypes, int count) {
    if (!tensors || !numel || !dtypes) return UHM_E_NULL;
    if (count <= 0) return UHM_E_SHAPE;
    long long chunks = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0) return UHM_E_SHAPE;
        if (numel[i] > (1LL << 56)) return UHM_E_TOO_LARGE;
        if (dtypes[i] < UHM_F32 || dtypes[i] > UHM_F16) return UHM_E_DTYPE;
        if (numel[i] && !tensors[i]) return UHM_E_NULL;
        if ((uintptr_t)tensors[i] & (elem_size(dtypes[i]) - 1)) return UHM_E_ALIGN;
        chunks += chunks_of(numel[i]);
        if (chunks > 0x7fffffffLL) return UHM_E_TOO_LARGE;
    }
    return 0;
}

// Bytes moved by both passes up to which the caches (256 MB of last-level cache) are left to hold the list.  Measured for the regressor's
// lists at 40 ... 128 px, three of them in turn, held / past the caches, us: clipping 107 MB 24.2 / 24.9, 165 MB 33.7 / 32.8,
// 236 MB 51.9 / 42.0; Adam 172 MB 37.2 / 39.1, 227 MB 47.4 / 46.8, 294 MB 62.3 / 56.7.
constexpr size_t CACHED = (size_t)192 << 20;

struct Span { uintptr_t begin, end; bool written; };

// whether memory that is written overlaps any other span
int check_spans(std::vector<Span>& spans) {
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
    uintptr_t any = 0, written = 0;
    for (const Span& s : spans) {
        if (s.begin < (s.written ? any : written)) return UHM_E_OVERLAP;
        any = std::max(any, s.end);
        if (s.written) written = std::max(written, s.end);
    }
    return 0;
}

// uhm_global_norm writes its workspace and the norm: neither may meet a tensor or the other.  (Tensors may overlap each other, so that
// they need not be put in order: 300 of them take 0.2 us.)
int check_norm_spans(const void* const* tensors, const long long* numel, const int* dtypes, int count, const float* norm, const void* workspace) {
    const uintptr_t n = (uintptr_t)norm, w = (uintptr_t)workspace, we = w + uhm_multi_workspace_bytes(count);
    if (n < we && w < n + sizeof(float)) return UHM_E_OVERLAP;
    for (int i = 0; i < count; ++i) {
        const uintptr_t t = (uintptr_t)tensors[i], te = t + (uintptr_t)numel[i] * elem_size(dtypes[i]);
        if (t < te && ((t < we && w < te) || (t < n + sizeof(float) && n < te))) return UHM_E_OVERLAP;
    }
    return 0;
}

// launches the first pass; *partials = how many sums it left
int sum_squares(const void* const* tensors, const long long* numel, const int* dtypes, int count, double* partial, int* partials,
                hipStream_t s) {
    int done = 0;
    const void* const* const lists[1] = {tensors};
    const int e = for_tables<NormTable, 1, 256>(lists, numel, dtypes, count, [&](const NormTable& t, unsigned grid) -> int {
        hipLaunchKernelGGL(sum_squares_kernel, dim3(grid), dim3(THREADS), 0, s, t, partial + done);
        done += (int)grid;
        return (int)hipGetLastError();
    });
    *partials = done;
    return e;
}

int check_workspace(const void* workspace, size_t bytes, int count) {
    if (!workspace || bytes < uhm_multi_workspace_bytes(count)) return UHM_E_WORKSPACE;
    return ((uintptr_t)workspace & 7) ? UHM_E_ALIGN : 0;
}

}  // namespace uhm

using namespace uhm;

extern "C" int uhm_abi_version(void) { return UHM_ABI_VERSION; }

extern "C" const char* uhm_error_string(int code) {
    switch (code) {
        case 0: return "ok";
        case UHM_E_NULL: return "UHM_E_NULL: a required pointer is NULL";
        case UHM_E_SHAPE: return "UHM_E_SHAPE: negative or inconsistent dimension, or an empty list";
        case UHM_E_WORKSPACE: return "UHM_E_WORKSPACE: workspace missing or too small";
        case UHM_E_TOO_LARGE: return "UHM_E_TOO_LARGE: a dimension is larger than the kernels index, or a 32-bit sum could overflow";
        case UHM_E_DTYPE: return "UHM_E_DTYPE: unknown element type";
        case UHM_E_OVERLAP: return "UHM_E_OVERLAP: memory that is written overlaps other memory of the call";
        case UHM_E_ALIGN: return "UHM_E_ALIGN: a pointer or stride is not aligned as required";
        case UHM_E_VALUE: return "UHM_E_VALUE: a scalar argument is outside its range";
        case UHM_E_HOST_MEMORY: return "UHM_E_HOST_MEMORY: out of host memory";
        default: return code > 0 ? hipGetErrorString((hipError_t)code) : "unknown uhm error";
    }
}

extern "C" size_t uhm_multi_workspace_bytes(int count) {
    if (count <= 0) return 0;
    return (size_t)((count + 255) / 256) * MAX_GRID * sizeof(double);
}

extern "C" int uhm_global_norm(const void* const* tensors, const long long* numel, const int* dtypes, int count, float* norm,
                               void* workspace, size_t workspace_bytes, uhm_stream_t stream) {
    if (!norm) return UHM_E_NULL;
    if (int e = check_list(tensors, numel, dtypes, count)) return e;
    if (int e = check_workspace(workspace, workspace_bytes, count)) return e;
    if (int e = check_norm_spans(tensors, numel, dtypes, count, norm, workspace)) return e;
    int partials = 0;
    if (int e = sum_squares(tensors, numel, dtypes, count, (double*)workspace, &partials, (hipStream_t)stream)) return e;
    hipLaunchKernelGGL(finish_norm_kernel, dim3(1), dim3(THREADS), 0, (hipStream_t)stream, (const double*)workspace, partials, norm);
    return (int)hipGetLastError();
}

extern "C" int uhm_clip_by_global_norm(const void* const* tensors, void* const* out, const long long* numel, const int* dtypes,
                                       int count, float clip_norm, const float* use_norm, float* norm, void* workspace,
                                       size_t workspace_bytes, uhm_stream_t stream) {
    if (!out) return UHM_E_NULL;
    if (int e = check_list(tensors, numel, dtypes, count)) return e;
    if (int e = check_list(out, numel, dtypes, count)) return e;
    if (!(clip_norm > 0.f)) return UHM_E_VALUE;
    if (!use_norm)
        if (int e = check_workspace(workspace, workspace_bytes, count)) return e;
    size_t touched = 0;
    try {
        std::vector<Span> spans;
        spans.reserve((size_t)count * 2 + 2);
        for (int i = 0; i < count; ++i) {
            const size_t bytes = (size_t)numel[i] * elem_size(dtypes[i]);
            if (!bytes) continue;
            touched += 3 * bytes;
            spans.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + bytes, true});
            if (out[i] != tensors[i]) spans.push_back({(uintptr_t)tensors[i], (uintptr_t)tensors[i] + bytes, false});
        }
        if (use_norm) spans.push_back({(uintptr_t)use_norm, (uintptr_t)use_norm + sizeof(float), false});
        else spans.push_back({(uintptr_t)workspace, (uintptr_t)workspace + uhm_multi_workspace_bytes(count), true});
        if (norm && norm != use_norm) spans.push_back({(uintptr_t)norm, (uintptr_t)norm + sizeof(float), true});
        if (int e = check_spans(spans)) return e;
    } catch (const std::bad_alloc&) {
        return UHM_E_HOST_MEMORY;
    }
    hipStream_t s = (hipStream_t)stream;
    int partials = 0;
    if (!use_norm)
        if (int e = sum_squares(tensors, numel, dtypes, count, (double*)workspace, &partials, s)) return e;
    bool told = false;
    const auto kernel = touched > CACHED ? scale_kernel<true> : scale_kernel<false>;
    const void* const* const lists[2] = {tensors, out};
    const int e = for_tables<ClipTable, 2, 128>(lists, numel, dtypes, count, [&](const ClipTable& t, unsigned grid) -> int {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), 0, s, t, (const double*)workspace, partials, use_norm, clip_norm,
                           told ? nullptr : norm);
        told = true;
        return (int)hipGetLastError();
    });
    if (e || told || !norm) return e;
    const ClipTable none{};                                    // a list of empty tensors: only the norm is written
    hipLaunchKernelGGL(kernel, dim3(1), dim3(THREADS), 0, s, none, (const double*)workspace, partials, use_norm, clip_norm, norm);
    return (int)hipGetLastError();
}

extern "C" int uhm_adam_clip_update(float* const* params, const void* const* grads, float* const* exp_avgs,
                                    float* const* exp_avg_sqs, const long long* numel, const int* grad_dtypes, int count,
                                    double lr, double beta1, double beta2, double eps, long long step, float clip_norm,
                                    unsigned flags, const float* use_norm, float* norm, void* workspace, size_t workspace_bytes, uhm_stream_t stream) {
    if (!params || !exp_avgs || !exp_avg_sqs) return UHM_E_NULL;
    if (int e = check_list(grads, numel, grad_dtypes, count)) return e;
    for (int i = 0; i < count; ++i) {
        if (!numel[i]) continue;
        if (!params[i] || !exp_avgs[i] || !exp_avg_sqs[i]) return UHM_E_NULL;
        if (((uintptr_t)params[i] | (uintptr_t)exp_avgs[i] | (uintptr_t)exp_avg_sqs[i]) & 3) return UHM_E_ALIGN;
    }
    if (!(clip_norm > 0.f) || step < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) ||
        !std::isfinite(eps) || !std::isfinite(lr) || (flags & ~UHM_SKIP_NONFINITE))
        return UHM_E_VALUE;
    if (!use_norm)
        if (int e = check_workspace(workspace, workspace_bytes, count)) return e;
    size_t touched = 0;
    try {
        std::vector<Span> spans;
        spans.reserve((size_t)count * 4 + 2);
        for (int i = 0; i < count; ++i) {
            if (!numel[i]) continue;
            const size_t bytes = (size_t)numel[i] * 4;
            touched += 6 * bytes + 2 * (size_t)numel[i] * elem_size(grad_dtypes[i]);
            for (uintptr_t p : {(uintptr_t)params[i], (uintptr_t)exp_avgs[i], (uintptr_t)exp_avg_sqs[i]}) spans.push_back({p, p + bytes, true});
            spans.push_back({(uintptr_t)grads[i], (uintptr_t)grads[i] + (size_t)numel[i] * elem_size(grad_dtypes[i]), false});
        }
        if (use_norm) spans.push_back({(uintptr_t)use_norm, (uintptr_t)use_norm + sizeof(float), false});
        else spans.push_back({(uintptr_t)workspace, (uintptr_t)workspace + uhm_multi_workspace_bytes(count), true});
        if (norm && norm != use_norm) spans.push_back({(uintptr_t)norm, (uintptr_t)norm + sizeof(float), true});
        if (int e = check_spans(spans)) return e;
    } catch (const std::bad_alloc&) {
        return UHM_E_HOST_MEMORY;
    }
    hipStream_t s = (hipStream_t)stream;
    int partials = 0;
    if (!use_norm)
        if (int e = sum_squares(grads, numel, grad_dtypes, count, (double*)workspace, &partials, s)) return e;
    // the scalars in f64, rounded once
    const double bias1 = 1.0 - std::pow(beta1, (double)step), bias2 = 1.0 - std::pow(beta2, (double)step);
    const AdamScalars a = {(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)(lr / bias1),
                           (float)(1.0 / std::sqrt(bias2)), (float)eps};
    const int skip = (flags & UHM_SKIP_NONFINITE) ? 1 : 0;
    bool told = false;
    const auto kernel = touched > CACHED ? adam_kernel<true> : adam_kernel<false>;
    const void* const* const lists[4] = {(const void* const*)params, grads, (const void* const*)exp_avgs, (const void* const*)exp_avg_sqs};
    const int e = for_tables<AdamTable, 4, 64>(lists, numel, grad_dtypes, count, [&](const AdamTable& t, unsigned grid) -> int {
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), 0, s, t, (const double*)workspace, partials, use_norm, clip_norm, skip, a,
                           told ? nullptr : norm);
        told = true;
        return (int)hipGetLastError();
    });
    if (e || told || !norm) return e;
    const AdamTable none{};                              // a list of empty tensors: only the norm is written
    hipLaunchKernelGGL(kernel, dim3(1), dim3(THREADS), 0, s, none, (const double*)workspace, partials, use_norm, clip_norm, skip, a, norm);
    return (int)hipGetLastError();
}
