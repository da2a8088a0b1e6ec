// uhm_int8.hip -- rows quantised to 8 bits and products of such rows (gfx950): the regressor's fully connected head in evaluation.
//
//   quantise:  top = max |x_r|, scale_r = top / 127, q = rne(x * (127 / top))
//   product :  out[m, n] = act(sum_k a[m, k] b[n, k] * sa[m] * sb[n] + bias[n])        exact 32-bit integer sums
//
// Up to FEW tokens: int8_few_kernel, which streams the weight once.  More: int8_matmul_kernel on v_mfma_i32_32x32x32_i8.  A block
// computes BM x BN outputs over a range of K.  Tiles of BK = 128 bytes of BM rows of a and BN rows of b go from memory straight
// into a ring of STAGES buffers in LDS; while one is multiplied the others are in flight (with 64 x 64 tiles two blocks of five
// buffers fill a CU's 160 KB: the loads of fc1 outrun the latency of HBM), with one barrier per tile.
// Few rows leave few tiles (fc1 at 64 pairs: 16 of 64 x 64): the K range is split over blocks, each writes its 32-bit sums to the
// workspace, and int8_join_kernel adds them (integers: the split does not change the result) and applies the epilogue.
//
// Measured on one MI355X (several sets of operands in turn, so that the weight comes from memory; passes among others):
//   fc1, 1024 x 32768:  1 pair 7.9 us (4.2 TB/s), from float 9.8; 64 pairs 11.2; 128 pairs from float 21.5 (quantising 6, product 11, join 3)
//   4096 x 4096 x 8192: 134 - 143 us with bf16 results, by card.  Where it takes 134, each 8192 of K more take 115 us = 2.4 POP/s; the loop without loads
//   takes 90 us, with neither loads nor LDS reads 69 us (the matrix instructions alone, at the clock that their power leaves): power, not latency.
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <type_traits>
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

// f32 of the integer sum (at most 2^31: one rounding), the two scales one after the other (their product alone could underflow).  The sum
// times a token's scale above LARGE could leave f32 where the result does not: there the channel's goes first.
constexpr float LARGE = 0x1p96f;
__device__ __forceinline__ float finish_in_order(int acc, float first, float second, float bias, int relu) {
    const float v = (float)acc * first * second + bias;
    return relu && v < 0.f ? 0.f : v;      // NaN stays
}
__device__ __forceinline__ float finish(int acc, float sa, float sb, float bias, int relu) {
    const bool large = fabsf(sa) > LARGE;
    return finish_in_order(acc, large ? sb : sa, large ? sa : sb, bias, relu);
}
__device__ __forceinline__ void put(void* out, int dtype, size_t at, float v) {
    if (dtype == UHM_F32) ((float*)out)[at] = v;
    else if (dtype == UHM_BF16) ((__bf16*)out)[at] = (__bf16)v;
    else ((_Float16*)out)[at] = (_Float16)v;
}

// the first `keep` of 4 and of 16 bytes, zeros behind them
__device__ __forceinline__ unsigned keep_first(unsigned w, int keep) {
    return keep >= 4 ? w : (keep <= 0 ? 0u : w & ((1u << (8 * keep)) - 1u));
}
__device__ __forceinline__ v4i keep_first(v4i v, int keep) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (int)keep_first((unsigned)v[j], keep - 4 * j);
    return v;
}
// the 16 bytes of a row from k on, zero behind K (one operand's zeros are enough for the product, the other's bytes may be anything)
__device__ __forceinline__ v4i load16(const int8_t* row, int k, int K, bool mask_tail) {
    v4i v = {0, 0, 0, 0};
    if (k < K) {
        v = *reinterpret_cast<const v4i*>(row + k);
        if (mask_tail) v = keep_first(v, K - k);
    }
    return v;
}

// Where a block works: its tile and its range of K.  Consecutive blocks go to the 8 XCDs in turn, each with an L2 of its own: the
// blocks of one XCD take a contiguous run of (K range, groups of 4 tile rows, tile columns), so that they share what they read.
struct Place { int m, n, z; };
__device__ __forceinline__ Place place(int mt, int nt, int splits) {
    const unsigned total = (unsigned)mt * nt * splits, q = total / 8, r = total % 8, xcd = blockIdx.x % 8;
    unsigned i = xcd * q + min(xcd, r) + blockIdx.x / 8;
    const unsigned z = i / ((unsigned)mt * nt);
    i -= z * mt * nt;
    const unsigned group = i / (4u * nt), rows = min(4u, mt - group * 4);
    i -= group * 4 * nt;
    return {(int)(group * 4 + i % rows), (int)(i / rows), (int)z};
}

template <int N> __device__ __forceinline__ void wait_for_loads() {          // ... but the last N, and every LDS read
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
}

template <int BM, int BN, int WM, int WN, int STAGES>      // WM x WN waves, each (BM / WM) x (BN / WN) outputs
__global__ __launch_bounds__(WM * WN * 64, 1) void int8_matmul_kernel(const int8_t* __restrict__ a, long long a_ld, const int8_t* __restrict__ b,
                                                                      long long b_ld, int M, int N, int K, int mt, int nt, int splits,
                                                                      int tiles_per_split, int* __restrict__ sums, const Epilogue e) {
    constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    // a tile's row is C chunks of 16 bytes; chunk c of row r sits at c ^ (r / PERIOD % C): 16 lanes that read one chunk of 16 rows at once
    // meet all 64 banks
    constexpr int C = BK / 16, PERIOD = 256 / BK, RL = 64 / C;         // RL: rows of one load of a wave
    constexpr int LA = BM / RL / WAVES, LB = BN / RL / WAVES;         // loads of a wave per tile
    static_assert(LA >= 1 && LB >= 1 && LA * WAVES * RL == BM && LB * WAVES * RL == BN, "staging");
    static_assert((WAVES * RL) % 16 == 0, "the chunk order of a load depends on its wave alone");
    __shared__ v4i sa[STAGES][BM * C], sb[STAGES][BN * C];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
    const Place at = place(mt, nt, splits);
    const long long m0 = (long long)at.m * BM, n0 = (long long)at.n * BN;
    const int t0 = at.z * tiles_per_split, t1 = min(t0 + tiles_per_split, (K + BK - 1) / BK), whole = min(t1, K / BK);

    // this lane's 16 bytes of each load: row lane / C, the chunk that belongs at position lane % C of it; rows behind the last one
    // repeat it (their outputs are not written)
    const int8_t* const base_a = a + m0 * a_ld;
    const int8_t* const base_b = b + n0 * b_ld;
    const unsigned chunk = ((lane % C) ^ ((wave * RL + lane / C) / PERIOD % C)) * 16;
    unsigned row_a[LA], row_b[LB];                                        // (256 rows of at most MAX_LD: 32 bits)
#pragma unroll
    for (int i = 0; i < LA; ++i) row_a[i] = (unsigned)min((long long)(i * WAVES + wave) * RL + lane / C, M - 1 - m0) * (unsigned)a_ld;
#pragma unroll
    for (int i = 0; i < LB; ++i) row_b[i] = (unsigned)min((long long)(i * WAVES + wave) * RL + lane / C, N - 1 - n0) * (unsigned)b_ld;
    auto to_lds = [](const int8_t* p, v4i* s) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p, (__attribute__((address_space(3))) void*)s, 16, 0, 0);
    };
    auto fetch = [&](int t, int buf) {
        const int k = t * BK;
        if (t < whole) {
#pragma unroll
            for (int i = 0; i < LA; ++i) to_lds(base_a + k + (row_a[i] + chunk), &sa[buf][(i * WAVES + wave) * 64]);
#pragma unroll
            for (int i = 0; i < LB; ++i) to_lds(base_b + k + (row_b[i] + chunk), &sb[buf][(i * WAVES + wave) * 64]);
        } else {                                                  // the tile that K ends in, through registers: zeros behind K
#pragma unroll
            for (int i = 0; i < LA; ++i) sa[buf][(i * WAVES + wave) * 64 + lane] = load16(base_a + row_a[i], k + chunk, K, true);
#pragma unroll
            for (int i = 0; i < LB; ++i) sb[buf][(i * WAVES + wave) * 64 + lane] = load16(base_b + row_b[i], k + chunk, K, false);
        }
    };

    v16i acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = v16i{};

    // The operands of a step are read before the matrix instructions of the step before it run, also across tiles: the last step of
    // a tile covers the barrier after which the next one may be read.  Behind it the tile's buffer is free and is filled again.
    constexpr int STEPS = BK / 32;
    static_assert(STEPS % 2 == 0, "two sets of operands");
    const int row = lane & 31, half = lane >> 5;
    v4i fa[2][TM], fb[2][TN];
    auto read = [&](int buf, int s) {
        const int c = (2 * s + half) ^ (row / PERIOD % C);
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[s & 1][i] = sa[buf][(wm + i * 32 + row) * C + c];
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[s & 1][j] = sb[buf][(wn + j * 32 + row) * C + c];
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
        if (t0 + i < t1) fetch(t0 + i, i);
    if (t0 + STAGES - 1 < whole) wait_for_loads<(LA + LB) * (STAGES - 1)>();
    else wait_for_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int buf = 0;
    if (t0 < t1) read(0, 0);
    for (int t = t0; t < t1; ++t) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s + 1 < STEPS) {
                read(buf, s + 1);
            } else if (t + 1 < t1) {
                // tile t + 1 is in LDS for every wave, and none still reads tile t
                if (t + STAGES - 1 < whole) wait_for_loads<(LA + LB) * (STAGES - 2)>();
                else wait_for_loads<0>();
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                const int next = buf + 1 == STAGES ? 0 : buf + 1;
                read(next, 0);
                if (t + STAGES < t1) fetch(t + STAGES, buf);
                buf = next;
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[s & 1][i], fb[s & 1][j], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // the tokens' scales through LDS: a load from memory for every row, one after the other, took 15 us of 4096 x 4096 outputs
    float* const scales = reinterpret_cast<float*>(&sa[0][0]);
    if (!sums) {
        __syncthreads();
        for (int i = tid; i < BM; i += WAVES * 64) scales[i] = e.a_scale[min(m0 + i, (long long)M - 1)];
        __syncthreads();
    }
    // D of a 32 x 32 tile: lane l, register i hold row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32
    auto each = [&](auto out) {
        float sbn[TN], bias[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const long long n = min(n0 + wn + j * 32 + row, (long long)N - 1);
            sbn[j] = sums ? 0.f : e.b_scale[n];
            bias[j] = sums || !e.bias ? 0.f : e.bias[n];
        }
        int m = wm + half * 4;
        size_t at = (size_t)(m0 + m) * N + n0 + wn + row;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                asm volatile("" : "+v"(m), "+v"(at));            // (a few rows' addresses at a time: all of them at once would spill)
                const float4 s4 = sums ? float4{} : *reinterpret_cast<const float4*>(scales + m);
                const float sam[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (m0 + m + k < M) {
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            if (n0 + wn + j * 32 + row < N) out(at + k * (size_t)N + j * 32, acc[i][j][4 * q + k], sam[k], sbn[j], bias[j]);
                    }
                m += 8;
                at += 8 * (size_t)N;
            }
    };
    // (whether a wave has a large scale among its rows is asked once: the choice at every output took 3 % of 2048 x 2048 x 2048)
    bool large = false;
    if (!sums)
#pragma unroll
        for (int r = 0; r < BM / WM; r += 64) large |= __any(fabsf(scales[wm + min(r + lane, BM / WM - 1)]) > LARGE);
    if (sums) {
        int* part = sums + (size_t)at.z * M * N;
        each([&](size_t at, int v, float, float, float) { part[at] = v; });
    } else if (large) {
        each([&](size_t at, int v, float sam, float sbn, float bias) { put(e.out, e.dtype, at, finish(v, sam, sbn, bias, e.relu)); });
    } else if (e.dtype == UHM_F32) {
        each([&](size_t at, int v, float sam, float sbn, float bias) { ((float*)e.out)[at] = finish_in_order(v, sam, sbn, bias, e.relu); });
    } else {
        each([&](size_t at, int v, float sam, float sbn, float bias) { put(e.out, e.dtype, at, finish_in_order(v, sam, sbn, bias, e.relu)); });
    }
}

// joins the splits: out[m, n] from sum_s sums[s][m][n].  The loads of 16 splits are in flight together (one after the other each
// waits for a trip to the L2 or beyond: 64 splits took 16 us that way).
__global__ __launch_bounds__(256) void int8_join_kernel(const int* __restrict__ sums, int splits, int M, int N, const Epilogue e) {
    const size_t total = (size_t)M * N;
    for (size_t at = (size_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (size_t)gridDim.x * 256) {
        const int m = (int)(at / N), n = (int)(at - (size_t)m * N);
        const float sam = e.a_scale[m], sbn = e.b_scale[n], bias = e.bias ? e.bias[n] : 0.f;
        int acc = 0;
        for (int s = 0; s < splits; s += 16) {
            int v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = s + j < splits ? sums[(size_t)(s + j) * total + at] : 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) acc += v[j];
        }
        put(e.out, e.dtype, at, finish(acc, sam, sbn, bias, e.relu));
    }
}

// ---- rows to 8 bits -----------------------------------------------------------------------------------------------------------
struct RowScale { float scale, inverse; };
// `bits`: the largest |x| as an integer (the order of non-negative floats; infinities and NaN are above all numbers)
__device__ __forceinline__ RowScale row_scale(unsigned bits) {
    if (bits >= 0x7f800000u) return {__builtin_nanf(""), 0.f};
    const float top = __uint_as_float(bits);
    if (top < 0x1p-120f) return {0.f, 0.f};              // 127 / top would leave the range of f32
    return {top / 127.0f, 127.0f / top};
}
// round to nearest even of the exact product: adding 1.5 * 2^23 leaves the integer in the low bits, with one rounding (fma)
__device__ __forceinline__ unsigned quantise(float x, RowScale s) {
    if (s.inverse == 0.f) return 0;
    return __float_as_uint(fmaf(x, s.inverse, 0x1.8p23f)) & 0xffu;
}
template <int T> struct Raw { using type = unsigned short; };
template <> struct Raw<UHM_F32> { using type = float; };
template <int T>
__device__ __forceinline__ float value(typename Raw<T>::type r) {
    if constexpr (T == UHM_F32) return r;
    else if constexpr (T == UHM_BF16) return __uint_as_float((unsigned)r << 16);
    else return __half2float(__ushort_as_half(r));
}
// Four elements of a row as they are in memory
template <int X> struct Four { typename Raw<X>::type v[4]; };
// COUNT times elements k .. k + 3, `step` elements apart.  Rows may start anywhere: the loads ask for no more than an element's
// alignment.  None has a branch, so that all are in flight: past K they give the row's last four again, which change no maximum.
template <int X, int COUNT>
__device__ __forceinline__ void load4s(Four<X> (&x)[COUNT], const void* row, int k, int step, int K) {
    using raw = typename Raw<X>::type;
    if (K >= 4) {                                                  // (the same for every thread)
#pragma unroll
        for (int i = 0; i < COUNT; ++i) x[i] = *reinterpret_cast<const Four<X>*>((const raw*)row + min(k + i * step, K - 4));
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i].v[j] = ((const raw*)row)[min(j, K - 1)];
    }
}
template <int X>
__device__ __forceinline__ unsigned top_of(const Four<X>& x) {
    unsigned t = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) t = max(t, __float_as_uint(value<X>(x.v[j])) & 0x7fffffffu);
    return t;
}
// elements k .. k + 3 (as load4s read them) in 8 bits, zeros behind K
template <int X>
__device__ __forceinline__ unsigned quantise4(const Four<X>& x, int k, int K, RowScale s) {
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) w |= quantise(value<X>(x.v[j]), s) << (8 * j);
    const int keep = K - k;                                        // of the group that K ends in, the last `keep` of four were read
    if (K >= 4 && keep < 4) w = keep <= 0 ? 0u : w >> (8 * (4 - keep));
    return keep_first(w, keep);
}

// the largest of `top` over a block of T threads, in every thread
template <int T>
__device__ __forceinline__ unsigned block_max(unsigned top) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d, 64));
    if constexpr (T > 64) {
        __shared__ unsigned sm[T / 64];
        if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < T / 64; ++w) top = max(top, sm[w]);
    }
    return top;
}

// One block per row.  Bound by the reads of x; a row of up to 32 T values stays in registers between the maximum and the rounding,
// a longer one is read a second time (out of the L2).  All of a thread's loads are in flight together.
template <int X, int T>
__global__ __launch_bounds__(T) void quantize_rows_kernel(const void* __restrict__ x, long long x_ld, int8_t* __restrict__ q,
                                                          long long q_ld, float* __restrict__ scale, int K) {
    constexpr int HELD = 8, SEGMENT = HELD * T * 4;
    const size_t row = blockIdx.x;
    const char* px = (const char*)x + row * x_ld * sizeof(typename Raw<X>::type);
    const int padded = (K + 15) & ~15, k0 = threadIdx.x * 4;
    Four<X> held[HELD];
    unsigned top = 0;
    for (int base = SEGMENT; base < K; base += SEGMENT) {
        load4s<X>(held, px, base + k0, T * 4, K);
#pragma unroll
        for (int i = 0; i < HELD; ++i) top = max(top, top_of(held[i]));
    }
    load4s<X>(held, px, k0, T * 4, K);
#pragma unroll
    for (int i = 0; i < HELD; ++i) top = max(top, top_of(held[i]));
    const RowScale s = row_scale(block_max<T>(top));
    if (threadIdx.x == 0) scale[row] = s.scale;
    int8_t* pq = q + row * q_ld;
    for (int base = 0; base < padded; base += SEGMENT) {
        if (base) load4s<X>(held, px, base + k0, T * 4, K);
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int k = base + k0 + i * T * 4;
            if (k < padded) *reinterpret_cast<unsigned*>(pq + k) = quantise4<X>(held[i], k, K, s);
        }
    }
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------------
// MB tokens: bound by the one read of the weight.  A block of T threads owns R channels and all of K (no split, no
// join, one launch): thread t holds bytes 16 t .. 16 t + 15 of every T * 16, AHEAD steps of every channel's row are in flight, products on
// the 4-way dot instruction (for so few tokens they take less time than the loads).  X < 0: tokens in 8 bits.  X >= 0: ONE token
// of that float type, quantised here: every block finds the row's maximum again (the row comes out of the L2) and keeps AHEAD
// steps of it in registers until then (what is longer is read again).
template <int T, int R, int MB, int X>
__global__ __launch_bounds__(T) void int8_few_kernel(const void* __restrict__ x, long long x_ld, const int8_t* __restrict__ b,
                                                     long long b_ld, int N, int K, const Epilogue e) {
    static_assert(X < 0 || MB == 1, "one token");
    constexpr int STEP = T * 16, AHEAD = 4;
    const int tid = threadIdx.x;
    const long long n0 = (long long)blockIdx.x * R;
    const int8_t* pb[R];
#pragma unroll
    for (int r = 0; r < R; ++r) pb[r] = b + min(n0 + r, (long long)N - 1) * b_ld;
    // a float token first: its maximum is found while the weight loads behind it are on their way (loads return in order).  Thread t
    // holds elements 4 t .. 4 t + 3 of every T * 4 -- consecutive lanes, consecutive memory: 16 elements a lane as the dot products
    // want them would take four times as many cycles per load (fc1: 5 us more) -- and hands them over in LDS, in 8 bits.
    constexpr int SEGMENT = AHEAD * STEP, HELD = X >= 0 ? SEGMENT / (T * 4) : 1;
    __shared__ v4i row8[X >= 0 ? SEGMENT / 16 : 1];
    Four<(X < 0 ? UHM_F32 : X)> held[HELD];
    if constexpr (X >= 0) {
        load4s<X>(held, x, tid * 4, T * 4, K);
        __builtin_amdgcn_sched_barrier(0);
    }
    // loads without a branch: past K the last 16 bytes again, which meet zeros of the token
    const int last = (K - 1) & ~15;
    v4i w[AHEAD][R];
    auto fetch = [&](int p, int k) {
#pragma unroll
        for (int r = 0; r < R; ++r) w[p][r] = *reinterpret_cast<const v4i*>(pb[r] + min(k, last));
    };
#pragma unroll
    for (int p = 0; p < AHEAD; ++p) fetch(p, p * STEP + tid * 16);

    RowScale s = {0.f, 0.f};
    const int8_t* px[MB];
    if constexpr (X >= 0) {
        __builtin_amdgcn_sched_barrier(0);
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < HELD; ++i) top = max(top, top_of(held[i]));
        for (int base = SEGMENT; base < K; base += SEGMENT) {
            Four<X> more[HELD];
            load4s<X>(more, x, base + tid * 4, T * 4, K);
#pragma unroll
            for (int i = 0; i < HELD; ++i) top = max(top, top_of(more[i]));
        }
        s = row_scale(block_max<T>(top));
    } else {
#pragma unroll
        for (int m = 0; m < MB; ++m) px[m] = (const int8_t*)x + m * x_ld;
    }

    int acc[R][MB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) acc[r][m] = 0;
    auto step = [&](int p, int k, const v4i (&xv)[MB]) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < MB; ++m)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][m] = __builtin_amdgcn_sdot4(w[p][r][j], xv[m][j], acc[r][m], false);
        if (k - tid * 16 + SEGMENT < K) fetch(p, k + SEGMENT);
    };
    for (int base = 0; base < K; base += SEGMENT) {
        if constexpr (X >= 0) {
            if (base) {
                load4s<X>(held, x, base + tid * 4, T * 4, K);      // (again, out of the L2)
                __syncthreads();                                   // everyone is through with the segment before
            }
#pragma unroll
            for (int i = 0; i < HELD; ++i) {
                const int k = base + (i * T + tid) * 4;
                reinterpret_cast<unsigned*>(row8)[i * T + tid] = quantise4<X>(held[i], k, K, s);
            }
            __syncthreads();
        }
#pragma unroll
        for (int p = 0; p < AHEAD; ++p) {
            const int k = base + p * STEP + tid * 16;
            v4i xv[MB];
            if constexpr (X >= 0) {
                xv[0] = row8[p * T + tid];
            } else {
#pragma unroll
                for (int m = 0; m < MB; ++m) xv[m] = *reinterpret_cast<const v4i*>(px[m] + min(k, last));
                if (base + (p + 1) * STEP > K) {                   // (the same for every thread)
#pragma unroll
                    for (int m = 0; m < MB; ++m) xv[m] = keep_first(xv[m], K - k);
                }
            }
            step(p, k, xv);
        }
    }

    constexpr int WAVES = T / 64;
    __shared__ int sm[WAVES][R * MB];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            int v = acc[r][m];
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
            if ((tid & 63) == 0) sm[tid >> 6][r * MB + m] = v;
        }
    __syncthreads();
    if (tid < R * MB) {
        const int r = tid / MB, m = tid % MB;
        const long long n = n0 + r;
        if (n < N) {
            int v = 0;
#pragma unroll
            for (int wv = 0; wv < WAVES; ++wv) v += sm[wv][tid];
            put(e.out, e.dtype, (size_t)m * N + n, finish(v, X >= 0 ? s.scale : e.a_scale[m], e.b_scale[n], e.bias ? e.bias[n] : 0.f, e.relu));
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
constexpr long long MAX_K = 131071, MAX_DIM = 0x7fffffffLL - 512;
constexpr long long MAX_LD = 1LL << 23;     // 256 rows of it are indexed in 32 bits
constexpr long long FEW = 2;               // tokens up to which int8_few_kernel reads the weight (fc1, replayed: 2 tokens 10.7 us, 4 12.5; tiles 12.2)

struct Plan { int bm, bn, splits, tiles_per_split; };

// The tile by how many of them there are, splits of K where they do not fill the 256 CUs.  Measured against the other tiles and splits on 19
// shapes, f32 results, replays of captured calls (about 1 us a launch more than passes among others): within 7 % of the best of each but for
// 128 x 1024 x 32768, 19.1 us at 16 splits | 16.7 at 8.  us, tile / splits taken | the other side:
//   32 x 128 up to 32 tokens:  16 x 1024 x 32768 12.5 at 32 splits | 12.3 at 16, 14.2 at 64
//   256 x 256 from 200 tiles:  4096 x 4096 x 8192 151 | 207 with 128 x 128; below, 1500 x 1500 x 3000 (36 of them) 27.5 | 56.5
//   128 x 128 from 200 tiles:  2048 x 2048 x 2048 23.6 | 27.1 with 64 x 64; below, 1024 x 1024 x 1024 (64 of them) 8.9 | 15.9
//   64 x 64:                   64 x 1024 x 32768 13.1 at 16 splits | 14.6 at 32, 15.7 at 8; 1000 x 300 x 6000 14.7 at 5 | 14.4 at 4, 17.5 at 8, 19.0 at 1
// At least 8 tiles of K per split (a block's first loads take as long as several tiles), 4 where there are few blocks anyway:
// 100 x 50 x 5000 8.2 at 10 | 7.9 at 16.
inline Plan plan_of(long long M, long long N, long long K) {
    const auto tiles_of = [&](int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    Plan p;
    long long most;                            // splits: past these the partial sums cost more than the blocks they add bring
    if (M <= 32) { p.bm = 32; p.bn = 128; most = 32; }
    else if (tiles_of(256, 256) >= 200) { p.bm = p.bn = 256; most = 1; }
    else if (tiles_of(128, 128) >= 200) { p.bm = p.bn = 128; most = 1; }
    else { p.bm = p.bn = 64; most = tiles_of(64, 64) <= 8 ? 32 : 16; }
    const long long tiles = tiles_of(p.bm, p.bn), kt = (K + BK - 1) / BK, least = tiles <= 16 ? 4 : 8;
    long long s = tiles < 256 ? 512 / tiles : 1;
    if (s > most) s = most;
    if (s > kt / least) s = kt / least;
    if (s < 1) s = 1;
    p.tiles_per_split = (int)((kt + s - 1) / s);
    p.splits = (int)((kt + p.tiles_per_split - 1) / p.tiles_per_split);
    return p;
}

int check_product(long long M, long long N, long long K) {
    if (M < 0 || N < 0 || K < 1) return UHM_E_SHAPE;
    if (K > MAX_K || M > MAX_DIM || N > MAX_DIM) return UHM_E_TOO_LARGE;
    // the grid is a line of blocks, fewer than 2^32 threads: at most 2^22 tiles of 32 x 64 (K is only split where they are few)
    if (N > (1LL << 27) || ((M + 31) / 32) * ((N + 63) / 64) > (1LL << 22)) return UHM_E_TOO_LARGE;
    return 0;
}

// the memory of a call, to find whether something that is written meets any of it
struct Memory {
    uintptr_t begin[6], end[6];
    int count = 0;
    void add(const void* p, size_t bytes) {
        if (!p) return;
        begin[count] = (uintptr_t)p;
        end[count++] = (uintptr_t)p + bytes;
    }
    bool meets(const void* p, size_t bytes) const {
        for (int i = 0; i < count; ++i)
            if (begin[i] < (uintptr_t)p + bytes && (uintptr_t)p < end[i]) return true;
        return false;
    }
};

// what the entry points for products check alike (x: the tokens, in 8 bits with a_scale or as floats without); *all: their operands and output
int check_operands(const void* x, int x_size, long long x_ld, const float* a_scale, const int8_t* b, long long b_ld, const float* b_scale, const float* bias,
                   const void* out, int out_dtype, long long M, long long N, long long K, unsigned flags, Memory* all) {
    if (int err = check_product(M, N, K)) return err;
    if (x_ld < K || b_ld < K) return UHM_E_SHAPE;
    if (N > 1 && b_ld > MAX_LD) return UHM_E_TOO_LARGE;
    if (out_dtype < UHM_F32 || out_dtype > UHM_F16) return UHM_E_DTYPE;
    if (flags & ~UHM_RELU) return UHM_E_VALUE;
    if (M == 0 || N == 0) return 0;
    if (!x || !b || !b_scale || !out) return UHM_E_NULL;
    if ((((uintptr_t)b | (uintptr_t)b_ld) & 15) || (((uintptr_t)b_scale | (uintptr_t)bias) & 3) || ((uintptr_t)out & (out_dtype == UHM_F32 ? 3 : 1)))
        return UHM_E_ALIGN;
    all->add(x, ((size_t)(M - 1) * x_ld + K) * x_size);
    all->add(a_scale, (size_t)M * 4);
    all->add(b, (size_t)(N - 1) * b_ld + K);
    all->add(b_scale, (size_t)N * 4);
    all->add(bias, (size_t)N * 4);
    const size_t written = (size_t)M * N * (out_dtype == UHM_F32 ? 4 : 2);
    if (all->meets(out, written)) return UHM_E_OVERLAP;
    all->add(out, written);
    return 0;
}

template <int X>
int quantize_rows(const void* x, long long x_ld, int8_t* q, long long q_ld, float* scale, long long rows, long long K, hipStream_t s) {
    // as few threads as hold the row in registers
    auto launch = [&](auto kernel, int threads) -> int {
        const long long most = (1LL << 31) / threads;                  // (a launch has fewer than 2^32 threads)
        for (long long r = 0; r < rows; r += most) {
            const long long n = rows - r < most ? rows - r : most;
            hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads), 0, s, (const char*)x + (size_t)r * x_ld * sizeof(typename Raw<X>::type), x_ld,
                               q + (size_t)r * q_ld, q_ld, scale + r, (int)K);
            if (int err = (int)hipGetLastError()) return err;
        }
        return 0;
    };
    if (K <= 2048) return launch(quantize_rows_kernel<X, 64>, 64);
    if (K <= 8192) return launch(quantize_rows_kernel<X, 256>, 256);
    return launch(quantize_rows_kernel<X, 1024>, 1024);
}

template <int MB, int X>
int launch_few(const void* x, long long x_ld, const int8_t* b, long long b_ld, int N, int K, const Epilogue& e, hipStream_t s) {
    auto launch = [&](auto kernel, int threads, int R) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(((long long)N + R - 1) / R)), dim3(threads), 0, s, x, x_ld, b, b_ld, N, K, e);
    };
    // threads by K (up to four steps of 16 bytes each, then loops), channels per block by N: at least a block for every CU before a block takes more
    auto rows = [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (N >= 1024) launch(int8_few_kernel<T, 4, MB, X>, T, 4);
        else if (N >= 512) launch(int8_few_kernel<T, 2, MB, X>, T, 2);
        else launch(int8_few_kernel<T, 1, MB, X>, T, 1);
    };
    if (K <= 4096) rows(std::integral_constant<int, 64>{});
    else if (K <= 16384) rows(std::integral_constant<int, 256>{});
    else rows(std::integral_constant<int, 512>{});
    return (int)hipGetLastError();
}

int product(const int8_t* a, long long a_ld, const int8_t* b, long long b_ld, long long M, long long N, long long K, const Epilogue& e, int* sums,
            hipStream_t s) {
    if (M == 1) return launch_few<1, -1>(a, a_ld, b, b_ld, (int)N, (int)K, e, s);
    if (M == FEW) return launch_few<2, -1>(a, a_ld, b, b_ld, (int)N, (int)K, e, s);
    const Plan p = plan_of(M, N, K);
    const int mt = (int)((M + p.bm - 1) / p.bm), nt = (int)((N + p.bn - 1) / p.bn);
    if (p.splits == 1) sums = nullptr;
    auto launch = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)mt * nt * p.splits), dim3(threads), 0, s, a, a_ld, b, b_ld, (int)M, (int)N, (int)K, mt, nt, p.splits,
                           p.tiles_per_split, sums, e);
    };
    if (p.bm == 32) launch(int8_matmul_kernel<32, 128, 1, 4, 4>, 256);
    else if (p.bm == 64) launch(int8_matmul_kernel<64, 64, 2, 2, 5>, 256);
    else if (p.bm == 128) launch(int8_matmul_kernel<128, 128, 2, 2, 4>, 256);
    else launch(int8_matmul_kernel<256, 256, 2, 4, 2>, 512);
    if (int err = (int)hipGetLastError()) return err;
    if (p.splits > 1) {
        const long long blocks = (M * N + 255) / 256;
        hipLaunchKernelGGL(int8_join_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, s, sums, p.splits, (int)M, (int)N, e);
        return (int)hipGetLastError();
    }
    return 0;
}

size_t sums_bytes(long long M, long long N, long long K) {
    if (M <= FEW) return 0;
    const Plan p = plan_of(M, N, K);
    return p.splits > 1 ? (size_t)p.splits * M * N * sizeof(int) : 0;
}

// workspace of a layer on float tokens: rows in 8 bits, their scales, the partial sums
struct LinearSpace { long long q_ld; size_t scale, sums, total; };
LinearSpace linear_space(long long M, long long N, long long K) {
    LinearSpace w;
    w.q_ld = (K + 127) / 128 * 128;                              // rows start on 128 bytes
    w.scale = (size_t)M * w.q_ld;
    w.sums = (w.scale + M * sizeof(float) + 127) / 128 * 128;
    w.total = w.sums + sums_bytes(M, N, K);
    return w;
}

int check_space(const void* workspace, size_t bytes, size_t need, const Memory& others) {
    if (!need) return 0;
    if (!workspace || bytes < need) return UHM_E_WORKSPACE;
    if ((uintptr_t)workspace & 15) return UHM_E_ALIGN;
    return others.meets(workspace, need) ? UHM_E_OVERLAP : 0;
}

}  // namespace uhm

using namespace uhm;

extern "C" int uhm_quantize_rows(const void* x, int dtype, long long x_ld, int8_t* q, long long q_ld, float* scale, long long rows,
                                 long long K, uhm_stream_t stream) {
    if (rows < 0 || K < 1 || x_ld < K || q_ld < K) return UHM_E_SHAPE;
    if (rows > MAX_DIM || K > MAX_DIM - 65536) return UHM_E_TOO_LARGE;      // (indexes go one segment past K)
    if (dtype < UHM_F32 || dtype > UHM_F16) return UHM_E_DTYPE;
    if (rows == 0) return 0;
    if (!x || !q || !scale) return UHM_E_NULL;
    if (((uintptr_t)q & 15) || (q_ld & 15) || ((uintptr_t)x & (dtype == UHM_F32 ? 3 : 1)) || ((uintptr_t)scale & 3)) return UHM_E_ALIGN;
    // (the last row of q is written up to K rounded up to 16)
    const uintptr_t xb = (uintptr_t)x, xe = xb + ((uintptr_t)(rows - 1) * x_ld + K) * (dtype == UHM_F32 ? 4 : 2), qb = (uintptr_t)q,
                    qe = qb + (uintptr_t)(rows - 1) * q_ld + (K + 15) / 16 * 16, sb = (uintptr_t)scale, se = sb + (uintptr_t)rows * 4;
    if ((qb < xe && xb < qe) || (sb < xe && xb < se) || (sb < qe && qb < se)) return UHM_E_OVERLAP;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == UHM_F32) return quantize_rows<UHM_F32>(x, x_ld, q, q_ld, scale, rows, K, s);
    if (dtype == UHM_BF16) return quantize_rows<UHM_BF16>(x, x_ld, q, q_ld, scale, rows, K, s);
    return quantize_rows<UHM_F16>(x, x_ld, q, q_ld, scale, rows, K, s);
}

extern "C" size_t uhm_int8_matmul_workspace_bytes(long long M, long long N, long long K) {
    if (check_product(M, N, K) || M == 0 || N == 0) return 0;
    return sums_bytes(M, N, K);
}

extern "C" int uhm_int8_matmul(const int8_t* a, long long a_ld, const float* a_scale, const int8_t* b, long long b_ld,
                               const float* b_scale, const float* bias, void* out, int out_dtype, long long M, long long N, long long K,
                               unsigned flags, void* workspace, size_t workspace_bytes, uhm_stream_t stream) {
    Memory all;
    if (int err = check_operands(a, 1, a_ld, a_scale, b, b_ld, b_scale, bias, out, out_dtype, M, N, K, flags, &all)) return err;
    if (M == 0 || N == 0) return 0;
    if (!a_scale) return UHM_E_NULL;
    if (M > 1 && a_ld > MAX_LD) return UHM_E_TOO_LARGE;
    if ((((uintptr_t)a | (uintptr_t)a_ld) & 15) || ((uintptr_t)a_scale & 3)) return UHM_E_ALIGN;
    if (int err = check_space(workspace, workspace_bytes, sums_bytes(M, N, K), all)) return err;
    const Epilogue e = {a_scale, b_scale, bias, out, out_dtype, (flags & UHM_RELU) ? 1 : 0};
    return product(a, a_ld, b, b_ld, M, N, K, e, (int*)workspace, (hipStream_t)stream);
}

extern "C" size_t uhm_int8_linear_workspace_bytes(long long M, long long N, long long K) {
    if (check_product(M, N, K) || M <= 1 || N == 0) return 0;
    return linear_space(M, N, K).total;
}

extern "C" int uhm_int8_linear(const void* x, int dtype, long long x_ld, const int8_t* b, long long b_ld, const float* b_scale,
                               const float* bias, void* out, long long M, long long N, long long K, unsigned flags, void* workspace,
                               size_t workspace_bytes, uhm_stream_t stream) {
    Memory all;
    if (int err = check_operands(x, dtype == UHM_F32 ? 4 : 2, x_ld, nullptr, b, b_ld, b_scale, bias, out, dtype, M, N, K, flags, &all)) return err;
    if (M == 0 || N == 0) return 0;
    if ((uintptr_t)x & (dtype == UHM_F32 ? 3 : 1)) return UHM_E_ALIGN;
    hipStream_t s = (hipStream_t)stream;
    Epilogue e = {nullptr, b_scale, bias, out, dtype, (flags & UHM_RELU) ? 1 : 0};
    if (M == 1) {
        if (dtype == UHM_F32) return launch_few<1, UHM_F32>(x, x_ld, b, b_ld, (int)N, (int)K, e, s);
        if (dtype == UHM_BF16) return launch_few<1, UHM_BF16>(x, x_ld, b, b_ld, (int)N, (int)K, e, s);
        return launch_few<1, UHM_F16>(x, x_ld, b, b_ld, (int)N, (int)K, e, s);
    }
    const LinearSpace w = linear_space(M, N, K);
    if (int err = check_space(workspace, workspace_bytes, w.total, all)) return err;
    int8_t* q = (int8_t*)workspace;
    float* scale = (float*)((char*)workspace + w.scale);
    if (int err = uhm_quantize_rows(x, dtype, x_ld, q, w.q_ld, scale, M, K, stream)) return err;
    e.a_scale = scale;
    return product(q, w.q_ld, b, b_ld, M, N, K, e, (int*)((char*)workspace + w.sums), s);
}
