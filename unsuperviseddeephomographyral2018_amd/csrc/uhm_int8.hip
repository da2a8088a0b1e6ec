// uhm_int8.hip -- rows quantised to 8 bits and products of such rows (gfx950): the regressor's fully connected head in evaluation.
//
//   quantise:  top = max |x_r|, scale_r = top / 127, q = rne(x * (127 / top))
//   product :  out[m, n] = act(sum_k a[m, k] b[n, k] * sa[m] * sb[n] + bias[n])        exact 32-bit integer sums
//
// One tiled kernel for every size, on v_mfma_i32_32x32x32_i8.  A block computes BM x BN outputs over a range of K: tiles of
// BK = 128 bytes of BM rows of a and BN rows of b go global -> registers -> LDS (two buffers; the next tile's loads are in flight
// while the present one is multiplied, one barrier per tile).  A tile row is 128 bytes = 8 chunks of 16; chunk c of row r sits at
// position c ^ (r & 7), so that the 8 rows that 8 lanes read at once (one chunk each) cover all 64 banks' 128 bytes, and so does
// a row that 8 lanes write.
// Few rows leave few tiles (fc1 at 64 pairs: 8 of 64 x 128): the K range is split over gridDim.z blocks, each writes its 32-bit
// sums to the workspace, and a second kernel adds them (integers: the split does not change the result) and applies the epilogue.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include "../../include/uh_model_ops.h"

namespace uhm {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr int BK = 128;                    // bytes of K per tile

struct Epilogue {
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    void* out;
    int dtype;
    int relu;
};

// f32 of the integer sum (at most 2^31: one rounding), the two scales one after the other (their product alone could underflow)
__device__ __forceinline__ float finish(int acc, float sa, float sb, float bias, int relu) {
    const float v = (float)acc * sa * sb + bias;
    return relu && v < 0.f ? 0.f : v;      // NaN stays
}
__device__ __forceinline__ void put(void* out, int dtype, size_t at, float v) {
    if (dtype == UHM_F32) ((float*)out)[at] = v;
    else if (dtype == UHM_BF16) ((__bf16*)out)[at] = (__bf16)v;
    else ((_Float16*)out)[at] = (_Float16)v;
}

// the 16 bytes of a row from k on, zero behind K (one operand's zeros are enough for the product, the other's bytes may be anything)
__device__ __forceinline__ v4i load16(const int8_t* row, long long k, long long K, bool mask_tail) {
    v4i v = {0, 0, 0, 0};
    if (k < K) {
        v = *reinterpret_cast<const v4i*>(row + k);
        if (mask_tail && K - k < 16) {
            const int keep = (int)(K - k);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int b = keep - 4 * j;                            // bytes of word j that count
                v[j] &= b >= 4 ? -1 : (b <= 0 ? 0 : (int)((1u << (8 * b)) - 1u));
            }
        }
    }
    return v;
}

template <int BM, int BN, int WM, int WN>      // WM x WN waves, each (BM / WM) x (BN / WN) outputs
__global__ __launch_bounds__(WM * WN * 64) void int8_matmul_kernel(const int8_t* __restrict__ a, long long a_ld, const int8_t* __restrict__ b,
                                                                   long long b_ld, int M, int N, int K, int tiles_per_split,
                                                                   int* __restrict__ sums, const Epilogue e) {
    constexpr int THREADS = WM * WN * 64, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int LA = BM * (BK / 16) / THREADS, LB = BN * (BK / 16) / THREADS;   // 16-byte chunks a thread stages
    static_assert(LA >= 1 && LB >= 1 && LA * THREADS == BM * 8 && LB * THREADS == BN * 8, "staging");
    __shared__ v4i sa[2][BM * 8], sb[2][BN * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    const long long m0 = (long long)blockIdx.y * BM, n0 = (long long)blockIdx.x * BN;
    const int ktiles = (K + BK - 1) / BK;
    const int t0 = blockIdx.z * tiles_per_split, t1 = min(t0 + tiles_per_split, ktiles);

    // this thread's chunks: rows behind the last one repeat it (their outputs are not written)
    const int8_t* pa[LA];
    const int8_t* pb[LB];
    int at_a[LA], at_b[LB];
    const int chunk = tid & 7;
#pragma unroll
    for (int i = 0; i < LA; ++i) {
        const int r = (tid >> 3) + i * (THREADS / 8);
        pa[i] = a + min(m0 + r, (long long)M - 1) * a_ld;
        at_a[i] = r * 8 + (chunk ^ (r & 7));
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
        const int r = (tid >> 3) + i * (THREADS / 8);
        pb[i] = b + min(n0 + r, (long long)N - 1) * b_ld;
        at_b[i] = r * 8 + (chunk ^ (r & 7));
    }
    v4i ra[LA], rb[LB];
    auto load = [&](int t) {
        const long long k = (long long)t * BK + chunk * 16;
#pragma unroll
        for (int i = 0; i < LA; ++i) ra[i] = load16(pa[i], k, K, true);
#pragma unroll
        for (int i = 0; i < LB; ++i) rb[i] = load16(pb[i], k, K, false);
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < LA; ++i) sa[buf][at_a[i]] = ra[i];
#pragma unroll
        for (int i = 0; i < LB; ++i) sb[buf][at_b[i]] = rb[i];
    };

    v16i acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v16i{};

    if (t0 < t1) {
        load(t0);
        store(0);
        if (t0 + 1 < t1) load(t0 + 1);
        __syncthreads();
        const int row = lane & 31, half = lane >> 5;
        for (int t = t0; t < t1; ++t) {
            const int buf = (t - t0) & 1;
#pragma unroll
            for (int s = 0; s < BK / 32; ++s) {
                v4i fa[TM], fb[TN];
                const int c = 2 * s + half;
#pragma unroll
                for (int i = 0; i < TM; ++i) { const int r = wm + i * 32 + row; fa[i] = sa[buf][r * 8 + (c ^ (r & 7))]; }
#pragma unroll
                for (int j = 0; j < TN; ++j) { const int r = wn + j * 32 + row; fb[j] = sb[buf][r * 8 + (c ^ (r & 7))]; }
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
            }
            if (t + 1 < t1) {
                store(buf ^ 1);                                  // everyone left this buffer before the last barrier
                if (t + 2 < t1) load(t + 2);
            }
            __syncthreads();
        }
    }

    // D of a 32 x 32 tile: lane l, register i hold row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32
    const int col = lane & 31, r4 = (lane >> 5) * 4;
    const bool split = sums != nullptr;
    int* part = sums + (size_t)blockIdx.z * M * N;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const long long n = n0 + wn + j * 32 + col;
        if (n >= N) continue;
        const float sbn = split ? 0.f : e.b_scale[n], bias = split || !e.bias ? 0.f : e.bias[n];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const long long m = m0 + wm + i * 32 + 8 * (k >> 2) + r4 + (k & 3);
                if (m >= M) continue;
                const size_t at = (size_t)m * N + n;
                if (split) part[at] = acc[i][j][k];
                else put(e.out, e.dtype, at, finish(acc[i][j][k], e.a_scale[m], sbn, bias, e.relu));
            }
    }
}

// joins the splits: out[m, n] from sum_s sums[s][m][n]
__global__ __launch_bounds__(256) void int8_join_kernel(const int* __restrict__ sums, int splits, int M, int N, const Epilogue e) {
    const size_t total = (size_t)M * N;
    for (size_t at = (size_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (size_t)gridDim.x * 256) {
        const int m = (int)(at / N), n = (int)(at - (size_t)m * N);
        int acc = 0;
        for (int s = 0; s < splits; ++s) acc += sums[s * total + at];
        put(e.out, e.dtype, at, finish(acc, e.a_scale[m], e.b_scale[n], e.bias ? e.bias[n] : 0.f, e.relu));
    }
}

// ---- rows to 8 bits -----------------------------------------------------------------------------------------------------------
template <int T>
__device__ __forceinline__ float value(const void* x, size_t i) {
    if constexpr (T == UHM_F32) return ((const float*)x)[i];
    else if constexpr (T == UHM_BF16) return __uint_as_float((unsigned)((const unsigned short*)x)[i] << 16);
    else return __half2float(__ushort_as_half(((const unsigned short*)x)[i]));
}

struct RowScale { float scale, inverse; };
// `bits`: the largest |x| as an integer (the order of non-negative floats; infinities and NaN are above all numbers)
__device__ __forceinline__ RowScale row_scale(unsigned bits) {
    if (bits >= 0x7f800000u) return {__builtin_nanf(""), 0.f};
    const float top = __uint_as_float(bits);
    if (top < 0x1p-120f) return {0.f, 0.f};              // 127 / top would leave the range of f32
    return {top / 127.0f, 127.0f / top};
}
// round to nearest even of the exact product: adding 1.5 * 2^23 leaves the integer in the low bits, with one rounding (fma)
__device__ __forceinline__ int quantise(float x, RowScale s) {
    if (s.inverse == 0.f) return 0;
    return (int)(__float_as_uint(fmaf(x, s.inverse, 0x1.8p23f)) & 0xffu);
}

template <int T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ x, long long x_ld, int8_t* __restrict__ q,
                                                            long long q_ld, float* __restrict__ scale, int K) {
    __shared__ unsigned sm[4];
    const size_t row = blockIdx.x;
    const char* px = (const char*)x + row * x_ld * (T == UHM_F32 ? 4 : 2);
    unsigned top = 0;
    for (int k = threadIdx.x; k < K; k += 256) top = max(top, __float_as_uint(value<T>(px, k)) & 0x7fffffffu);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d, 64));
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = top;
    __syncthreads();
    const RowScale s = row_scale(max(max(sm[0], sm[1]), max(sm[2], sm[3])));
    if (threadIdx.x == 0) scale[row] = s.scale;
    int8_t* pq = q + row * q_ld;
    for (int k = threadIdx.x * 4; k < (K + 15) / 16 * 16; k += 1024) {
        unsigned w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < K) w |= (unsigned)quantise(value<T>(px, k + j), s) << (8 * j);
        *reinterpret_cast<unsigned*>(pq + k) = w;
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
constexpr long long MAX_K = 131071, MAX_DIM = 0x7fffffffLL - 512;

struct Plan { int bm, bn, splits, tiles_per_split; };

// v1 rule: the tile follows M; K is split until about 512 blocks run, each keeping at least 4 tiles of K
inline Plan plan_of(long long M, long long N, long long K) {
    Plan p;
    if (M <= 32) { p.bm = 32; p.bn = 128; }
    else if (M <= 64) { p.bm = 64; p.bn = 128; }
    else { p.bm = 128; p.bn = 128; }
    if (((M + 255) / 256) * ((N + 255) / 256) >= 200) p.bm = p.bn = 256;
    const long long tiles = ((M + p.bm - 1) / p.bm) * ((N + p.bn - 1) / p.bn), kt = (K + BK - 1) / BK;
    long long s = 1;
    if (tiles < 256) s = 512 / tiles;
    if (s > kt / 4) s = kt / 4;
    if (s < 1) s = 1;
    p.tiles_per_split = (int)((kt + s - 1) / s);
    p.splits = (int)((kt + p.tiles_per_split - 1) / p.tiles_per_split);
    return p;
}

int check_product(long long M, long long N, long long K) {
    if (M < 0 || N < 0 || K < 1) return UHM_E_SHAPE;
    if (K > MAX_K || M > MAX_DIM || N > MAX_DIM) return UHM_E_TOO_LARGE;
    // grid: blocks along M in gridDim.y, sizes of the output in 64 bits
    if ((M + 31) / 32 > 65535) return UHM_E_TOO_LARGE;
    return 0;
}

}  // namespace uhm

using namespace uhm;

extern "C" int uhm_quantize_rows(const void* x, int dtype, long long x_ld, int8_t* q, long long q_ld, float* scale, long long rows,
                                 long long K, uhm_stream_t stream) {
    if (rows < 0 || K < 1 || x_ld < K || q_ld < K) return UHM_E_SHAPE;
    if (rows > MAX_DIM || K > MAX_DIM) return UHM_E_TOO_LARGE;
    if (dtype < UHM_F32 || dtype > UHM_F16) return UHM_E_DTYPE;
    if (rows == 0) return 0;
    if (!x || !q || !scale) return UHM_E_NULL;
    if (((uintptr_t)q & 15) || (q_ld & 15) || ((uintptr_t)x & (dtype == UHM_F32 ? 3 : 1)) || ((uintptr_t)scale & 3)) return UHM_E_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)rows), block(256);
    if (dtype == UHM_F32) hipLaunchKernelGGL(quantize_rows_kernel<UHM_F32>, grid, block, 0, s, x, x_ld, q, q_ld, scale, (int)K);
    else if (dtype == UHM_BF16) hipLaunchKernelGGL(quantize_rows_kernel<UHM_BF16>, grid, block, 0, s, x, x_ld, q, q_ld, scale, (int)K);
    else hipLaunchKernelGGL(quantize_rows_kernel<UHM_F16>, grid, block, 0, s, x, x_ld, q, q_ld, scale, (int)K);
    return (int)hipGetLastError();
}

extern "C" size_t uhm_int8_matmul_workspace_bytes(long long M, long long N, long long K) {
    if (check_product(M, N, K) || M == 0 || N == 0) return 0;
    const Plan p = plan_of(M, N, K);
    return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(int) : 0;
}

extern "C" int uhm_int8_matmul(const int8_t* a, long long a_ld, const float* a_scale, const int8_t* b, long long b_ld,
                               const float* b_scale, const float* bias, void* out, int out_dtype, long long M, long long N, long long K,
                               unsigned flags, void* workspace, size_t workspace_bytes, uhm_stream_t stream) {
    if (int err = check_product(M, N, K)) return err;
    if (a_ld < K || b_ld < K) return UHM_E_SHAPE;
    if (out_dtype < UHM_F32 || out_dtype > UHM_F16) return UHM_E_DTYPE;
    if (flags & ~UHM_RELU) return UHM_E_VALUE;
    if (M == 0 || N == 0) return 0;
    if (!a || !a_scale || !b || !b_scale || !out) return UHM_E_NULL;
    if ((((uintptr_t)a | (uintptr_t)b | (uintptr_t)a_ld | (uintptr_t)b_ld) & 15) ||
        (((uintptr_t)a_scale | (uintptr_t)b_scale | (uintptr_t)bias) & 3) || ((uintptr_t)out & (out_dtype == UHM_F32 ? 3 : 1)))
        return UHM_E_ALIGN;
    const Plan p = plan_of(M, N, K);
    int* sums = nullptr;
    if (p.splits > 1) {
        if (!workspace || workspace_bytes < uhm_int8_matmul_workspace_bytes(M, N, K)) return UHM_E_WORKSPACE;
        if ((uintptr_t)workspace & 15) return UHM_E_ALIGN;
        sums = (int*)workspace;
    }
    const Epilogue e = {a_scale, b_scale, bias, out, out_dtype, (flags & UHM_RELU) ? 1 : 0};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid((unsigned)((N + p.bn - 1) / p.bn), (unsigned)((M + p.bm - 1) / p.bm), (unsigned)p.splits);
    auto launch = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, a, a_ld, b, b_ld, (int)M, (int)N, (int)K, p.tiles_per_split, sums, e);
    };
    if (p.bm == 32) launch(int8_matmul_kernel<32, 128, 1, 4>, 256);
    else if (p.bm == 64) launch(int8_matmul_kernel<64, 128, 2, 2>, 256);
    else if (p.bm == 128) launch(int8_matmul_kernel<128, 128, 2, 2>, 256);
    else launch(int8_matmul_kernel<256, 256, 2, 4>, 512);
    if (int err = (int)hipGetLastError()) return err;
    if (p.splits > 1) {
        const long long blocks = (M * N + 255) / 256;
        hipLaunchKernelGGL(int8_join_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, sums, p.splits, (int)M, (int)N, e);
        return (int)hipGetLastError();
    }
    return 0;
}
