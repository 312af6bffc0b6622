// Row-wise building blocks of the classifier-head kernels (layernorm.hip, scores.hip, distill.hip): 16-byte pieces of rows in
// fp32 / bf16 / fp16, held packed in registers, and reductions over the G threads ("team") that share a row.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

#define WFD_F32 0
#define WFD_BF16 1
#define WFD_F16 2

static inline float log2e_over(float t) { return (float)(1.4426950408889634 / (double)t); }
static inline bool wfd_dtype_ok(int t) { return t >= WFD_F32 && t <= WFD_F16; }

static inline int elems_of(int dtype) { return dtype == WFD_F32 ? 4 : 8; }     // of one 16-byte piece
static inline bool rows_ok(const void* p, int ld, int M, int N, int dtype) {
    const uintptr_t align = dtype == WFD_F32 ? 3 : 1;
    return p && !((uintptr_t)p & align) && (M <= 1 || ld >= N);
}
// one buffer under two row strides would be written before it is read
static inline bool same_rows(const void* out, int ldo, const void* in, int ldi, int M) { return out != in || ldo == ldi || M <= 1; }
// a launch counts its threads in 32 bits
static inline bool launchable(long blocks, int threads) { return blocks * threads <= 0xffffffffL; }

__device__ __forceinline__ int cdiv_dev(int a, int b) { return (a + b - 1) / b; }

template <class T> struct Pack { static constexpr int N = 16 / (int)sizeof(T); };   // elements of one 16-byte piece

// Rows begin wherever their stride puts them (an odd width of 16-bit values leaves every second row off even a 4-byte border):
// gfx950 serves 16-byte accesses at any address, so pieces are counted from the row's first element, unaligned.  The n % N elements
// behind the last whole piece go one to a thread.  An address off a 4-byte border costs a tenth of a long read's rate (4096 rows of
// 50257 bf16: 90.7 us, 50258: 76.8, 50264: 76.4), so long rows leave out their first element there and count from the second.
struct __attribute__((packed, aligned(2))) Raw16u { unsigned v[4]; };
struct Raw16 { unsigned v[4]; };

template <class T> __device__ __forceinline__ Raw16 load16(const T* p) {
    Raw16u r = *reinterpret_cast<const Raw16u*>(p);
    return Raw16{{r.v[0], r.v[1], r.v[2], r.v[3]}};
}
template <class T> __device__ __forceinline__ void store16(T* p, const Raw16& r) {
    *reinterpret_cast<Raw16u*>(p) = Raw16u{{r.v[0], r.v[1], r.v[2], r.v[3]}};
}

// A result that the 256 MiB of last-level cache cannot hold until its reader comes is better written past the caches; a smaller one
// is not.  The gradient of `rows` x 32000 bf16 scores and a sum that reads it, us in the caches / past them: 96 MB 73 / 88, 192 MB
// 148 / 161, 224 MB 182 / 185, 256 MB 214 / 210, 288 MB 246 / 235 (the gradient alone: 40 / 36, 73 / 70, 85 / 81, 96 / 92, 109 / 104).
constexpr long LAST_LEVEL = 250000000;
static inline bool past_caches(long rows, long n, int bytes) { return rows * n * bytes >= LAST_LEVEL; }
template <class T> __device__ __forceinline__ void store16(T* p, const Raw16& r, bool past) {
    typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(2)));
    if (past) __builtin_nontemporal_store(u4{r.v[0], r.v[1], r.v[2], r.v[3]}, reinterpret_cast<u4*>(p));
    else store16(p, r);
}

// 1 where a row of 16-bit values begins between two 4-byte borders
template <class T> __device__ __forceinline__ int off_border(const T* p) {
    return sizeof(T) == 2 ? (int)((uintptr_t)p >> 1 & 1) : 0;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return (float)v; }
__device__ __forceinline__ float to_f32(f16_t v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }    // round to nearest even

// element e of a packed piece (e is a constant after unrolling)
template <class T> __device__ __forceinline__ float elem(const Raw16& r, int e);
template <> __device__ __forceinline__ float elem<float>(const Raw16& r, int e) { return __uint_as_float(r.v[e]); }
template <> __device__ __forceinline__ float elem<bf16_t>(const Raw16& r, int e) {
    return __uint_as_float((e & 1) ? (r.v[e >> 1] & 0xffff0000u) : (r.v[e >> 1] << 16));
}
template <> __device__ __forceinline__ float elem<f16_t>(const Raw16& r, int e) {
    const unsigned short h = (unsigned short)((e & 1) ? r.v[e >> 1] >> 16 : r.v[e >> 1] & 0xffffu);
    return (float)__builtin_bit_cast(_Float16, h);
}

template <class T> __device__ __forceinline__ Raw16 pack(const float* f) {
    Raw16 r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) r.v[e] = __float_as_uint(f[e]);
    } else {
        typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const t2 h = {(T)f[2 * e], (T)f[2 * e + 1]};
            __builtin_memcpy(&r.v[e], &h, 4);
        }
    }
    return r;
}

// Hides from the compiler that a packed piece has been unpacked before: it would otherwise keep the unpacked values of one
// phase alive for the next, at twice the registers (and spills where a thread holds 16 pieces).
__device__ __forceinline__ void keep_packed(Raw16& r) {
    asm volatile("" : "+v"(r.v[0]), "+v"(r.v[1]), "+v"(r.v[2]), "+v"(r.v[3]));
}

// the raw pattern of `fill` in every element
template <class T> __device__ __forceinline__ unsigned raw_fill(float fill) {
    float f[8] = {fill, fill, fill, fill, fill, fill, fill, fill};
    return pack<T>(f).v[0];
}

// A team's pieces: thread t of G has pieces r * G + t of a row's P whole ones.  A load under a condition with another value beside it
// makes the compiler wait for each one before the next (it merges registers behind the branch), so a thread without a piece reads
// the row's last one instead, and `only` puts the value of an empty place where the piece is used.  ONE: the team of the shortest
// rows, which may have no whole piece at all and only has the one load to wait for.
template <class T, bool ONE> __device__ __forceinline__ void team_load(Raw16& d, const T* row, int piece, int P) {
    if constexpr (ONE) {
        d = Raw16{{0u, 0u, 0u, 0u}};
        if (piece < P) d = load16(row + piece * Pack<T>::N);
    } else {
        d = load16(row + min(piece, P - 1) * Pack<T>::N);
    }
}
__device__ __forceinline__ void only(Raw16& d, bool here, unsigned none) {
#pragma unroll
    for (int i = 0; i < 4; ++i) d.v[i] = here ? d.v[i] : none;
}

// elements [i0, i0 + Pack<T>::N) of a row of n; those past the end read as `fill`
template <class T> __device__ __forceinline__ Raw16 load_piece(const T* row, int i0, int n, float fill) {
    constexpr int E = Pack<T>::N;
    if (i0 + E <= n) return load16(row + i0);
    float f[8];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = i0 + e < n ? to_f32(row[i0 + e]) : fill;
    return pack<T>(f);
}
template <class T> __device__ __forceinline__ void store_piece(T* row, int i0, int n, const float* f, bool past = false) {
    constexpr int E = Pack<T>::N;
    if (i0 + E <= n) {
        store16(row + i0, pack<T>(f), past);
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (i0 + e < n) row[i0 + e] = from_f32<T>(f[e]);
}

// ---- reductions over the lanes of a wave: DPP inside 16 lanes (no LDS latency), two lane exchanges above ----------------
// Every step adds a pair in both of its lanes, so all lanes end with the same bits -- as long as neither addition is fused with the
// product that made the lane's own value: contraction is off in the sums.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lanes_sum16(float v) {
#pragma clang fp contract(off)
    v += dpp<0xB1>(v);      // quad_perm 1,0,3,2
    v += dpp<0x4E>(v);      // quad_perm 2,3,0,1
    v += dpp<0x141>(v);     // row_half_mirror
    v += dpp<0x140>(v);     // row_mirror
    return v;
}
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const int2 w = __builtin_bit_cast(int2, v);
    return __builtin_bit_cast(double, int2{__builtin_amdgcn_update_dpp(0, w.x, CTRL, 0xf, 0xf, true),
                                           __builtin_amdgcn_update_dpp(0, w.y, CTRL, 0xf, 0xf, true)});
}
template <int G> __device__ __forceinline__ double lanes_sum(double v) {
#pragma clang fp contract(off)
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}
__device__ __forceinline__ float lanes_max16(float v) {
    v = fmaxf(v, dpp<0xB1>(v));
    v = fmaxf(v, dpp<0x4E>(v));
    v = fmaxf(v, dpp<0x141>(v));
    v = fmaxf(v, dpp<0x140>(v));
    return v;
}
template <int G> __device__ __forceinline__ float lanes_sum(float v) {
#pragma clang fp contract(off)
    v = lanes_sum16(v);
    if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}
template <int G> __device__ __forceinline__ float lanes_max(float v) {
    v = lanes_max16(v);
    if constexpr (G >= 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
    if constexpr (G >= 64) v = fmaxf(v, __shfl_xor(v, 32, 64));
    return v;
}

// Two sums over a team of G threads; G <= 64 stays inside the wave, above it the wave sums meet in `slot` (2 * G / 64 floats of
// LDS that nothing else touches until the next barrier after this one) and are added in wave order by every thread.
template <int G> __device__ __forceinline__ float2 team_sum2(float a, float b, float* slot) {
    a = lanes_sum<(G < 64 ? G : 64)>(a);
    b = lanes_sum<(G < 64 ? G : 64)>(b);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) { slot[2 * w] = a; slot[2 * w + 1] = b; }
        __syncthreads();
        a = 0.f; b = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) { a += slot[2 * i]; b += slot[2 * i + 1]; }
    }
    return make_float2(a, b);
}
template <int G> __device__ __forceinline__ float team_sum(float a, float* slot) {
    a = lanes_sum<(G < 64 ? G : 64)>(a);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slot[w] = a;
        __syncthreads();
        a = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) a += slot[i];
    }
    return a;
}
template <int G> __device__ __forceinline__ float team_max(float a, float* slot) {
    a = lanes_max<(G < 64 ? G : 64)>(a);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) slot[w] = a;
        __syncthreads();
        a = slot[0];
#pragma unroll
        for (int i = 1; i < W; ++i) a = fmaxf(a, slot[i]);
    }
    return a;
}

// ---- sums of exponentials about a maximum --------------------------------------------------------------------------------
// exp((x - m) / T) = 2^((x - m) c), c = log2(e) / T.  The scores take the difference first: the maximum itself then gives 1 to the bit,
// so a class alone in its row has log probability 0.  Distillation, whose gradient has two exponentials per element, takes
// 2^(x c - m c): one fused multiply-add with the rounded R = m c (3000 x 70000 fp16 197 us, difference first 210), and what R's rounding
// leaves (m c - R, exact by fma) is taken out of a whole group's sum at once.  Where m c is so large that the remainder would be
// no small exponent itself (rows at the type's lowest value, whose product may even leave fp32's range) the difference comes first.
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float LOWEST = -3.402823466e38f;       // floor of a maximum: x - m stays defined for rows of nothing but -inf
constexpr float FAINT = -1e4f;                   // an exponent whose exponential is 0: stands in where 0 * -inf would be NaN
constexpr float WIDE = 1e6f;                     // m c from which on: the remainder stays below 2^-24 * 1e6 = 0.06

__device__ __forceinline__ float exp2_of(float v) { return __builtin_amdgcn_exp2f(v); }
