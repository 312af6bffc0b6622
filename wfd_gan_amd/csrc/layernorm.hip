// Layer norm over the last dimension, forward and backward, fp32 / bf16 / fp16 rows with weights of the same type or fp32.
//   forward   mean = sum x / N,  rstd = 1 / sqrt(sum (x - mean)^2 / N + eps),  y = (x - mean) rstd w + b
//   backward  xh = (x - mean) rstd,  v = dy w:
//             dx = rstd (v - sum v / N - xh sum(v xh) / N),  dw = sum_rows dy xh,  db = sum_rows dy
// Bound by memory: forward reads and writes a row once, backward reads two and writes one.  A row is held packed in the registers
// of its team (16 / 64 / 256 / 1024 threads), so the variance is the two-pass one about the true mean and costs no second read.
#include "rowops.h"

namespace {

struct LnFwd {
    const void* X;
    const void* W;
    const void* B;
    void* Y;
    float* mean;
    float* rstd;
    int ldx, ldy, M, N;
    float eps;
};
struct LnBwd {
    const void* DY;
    const void* X;
    const void* W;
    const float* mean;
    const float* rstd;
    void* DX;
    float* part;       // [blocks][2][N]: each workgroup's sums of dy xh and dy
    int lddy, ldx, lddx, M, N;
};

template <class WT, int E> __device__ __forceinline__ void load_weights(float* f, const WT* w, int i0, int n, float none) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = none;
    if (!w) return;
    constexpr int P = Pack<WT>::N;
    if (i0 + E <= n) {
        if constexpr (P >= E) {
            const Raw16 r = load16(w + i0);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = elem<WT>(r, e);
        } else {
#pragma unroll
            for (int h = 0; h < E / P; ++h) {
                const Raw16 r = load16(w + i0 + h * P);
#pragma unroll
                for (int e = 0; e < P; ++e) f[h * P + e] = elem<WT>(r, e);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (i0 + e < n) f[e] = to_f32(w[i0 + e]);
    }
}

// ---- forward: a team of G threads per row, R pieces per thread in registers -----------------------------------------
template <class T, class WT, int G, int R>
__global__ __launch_bounds__(G < 256 ? 256 : G) void ln_fwd_kernel(LnFwd g) {
    constexpr int E = Pack<T>::N, TEAMS = G < 256 ? 256 / G : 1;
    __shared__ float slot[2][G > 64 ? G / 64 : 1];
    const int t = threadIdx.x % G;
    const long row = (long)blockIdx.x * TEAMS + threadIdx.x / G;
    if (row >= g.M) return;                              // whole teams; only teams of at most one wave share a workgroup
    const T* x = (const T*)g.X + row * g.ldx;
    const int N = g.N;
    Raw16 d[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i0 = (r * G + t) * E;
        if (i0 < N) d[r] = load_piece(x, i0, N, 0.f);
    }
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if ((r * G + t) * E < N)
#pragma unroll
            for (int e = 0; e < E; ++e) s += elem<T>(d[r], e);
    const float mean = team_sum<G>(s, slot[0]) / (float)N;
    float q = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i0 = (r * G + t) * E;
        if (i0 < N)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float c = i0 + e < N ? elem<T>(d[r], e) - mean : 0.f;
                q = fmaf(c, c, q);
            }
    }
    const float rstd = 1.f / sqrtf(team_sum<G>(q, slot[1]) / (float)N + g.eps);
    if (t == 0) {
        if (g.mean) g.mean[row] = mean;
        if (g.rstd) g.rstd[row] = rstd;
    }
    T* y = (T*)g.Y + row * g.ldy;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i0 = (r * G + t) * E;
        if (i0 < N) {
            float w[E], b[E], o[E];
            load_weights<WT, E>(w, (const WT*)g.W, i0, N, 1.f);
            load_weights<WT, E>(b, (const WT*)g.B, i0, N, 0.f);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf((elem<T>(d[r], e) - mean) * rstd, w[e], b[e]);
            store_piece(y, i0, N, o);
        }
    }
}

// rows longer than a workgroup's registers hold: three walks over the row (the second and third from the caches)
template <class T, class WT> __global__ __launch_bounds__(1024) void ln_fwd_long_kernel(LnFwd g) {
    constexpr int E = Pack<T>::N, G = 1024;
    __shared__ float slot[2][G / 64];
    const long row = blockIdx.x;
    const int t = threadIdx.x, N = g.N;
    const T* x = (const T*)g.X + row * g.ldx;
    float s = 0.f;
    for (long i0 = (long)t * E; i0 < N; i0 += G * E) {
        const Raw16 d = load_piece(x, (int)i0, N, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) s += elem<T>(d, e);
    }
    const float mean = team_sum<G>(s, slot[0]) / (float)N;
    float q = 0.f;
    for (long i0 = (long)t * E; i0 < N; i0 += G * E) {
        const Raw16 d = load_piece(x, (int)i0, N, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float c = i0 + e < N ? elem<T>(d, e) - mean : 0.f;
            q = fmaf(c, c, q);
        }
    }
    const float rstd = 1.f / sqrtf(team_sum<G>(q, slot[1]) / (float)N + g.eps);
    if (t == 0) {
        if (g.mean) g.mean[row] = mean;
        if (g.rstd) g.rstd[row] = rstd;
    }
    T* y = (T*)g.Y + row * g.ldy;
    for (long i0 = (long)t * E; i0 < N; i0 += G * E) {
        const Raw16 d = load_piece(x, (int)i0, N, 0.f);
        float w[E], b[E], o[E];
        load_weights<WT, E>(w, (const WT*)g.W, (int)i0, N, 1.f);
        load_weights<WT, E>(b, (const WT*)g.B, (int)i0, N, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf((elem<T>(d, e) - mean) * rstd, w[e], b[e]);
        store_piece(y, (int)i0, N, o);
    }
}

// ---- backward: a team walks rows, its threads keep the sums of dy xh and dy of their columns in registers ---------------
template <class T, class WT, int G, int R>
__global__ __launch_bounds__(G < 256 ? 256 : G) void ln_bwd_kernel(LnBwd g) {
    constexpr int E = Pack<T>::N, TEAMS = G < 256 ? 256 / G : 1, W = G > 64 ? G / 64 : 1;
    __shared__ float slot[2][2 * W];
    const int t = threadIdx.x % G, team = threadIdx.x / G, N = g.N;
    float w[R][E], sw[R][E], sb[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i0 = (r * G + t) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) { sw[r][e] = 0.f; sb[r][e] = 0.f; w[r][e] = 0.f; }
        if (i0 < N) load_weights<WT, E>(w[r], (const WT*)g.W, i0, N, 1.f);
    }
    const float inv = 1.f / (float)N;
    int par = 0;
    for (long row = (long)blockIdx.x * TEAMS + team; row < g.M; row += (long)gridDim.x * TEAMS, par ^= 1) {
        const T* x = (const T*)g.X + row * g.ldx;
        const T* dy = (const T*)g.DY + row * g.lddy;
        const float mean = g.mean[row], rstd = g.rstd[row];
        Raw16 dx_[R], dd[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i0 = (r * G + t) * E;
            if (i0 < N) {
                dx_[r] = load_piece(x, i0, N, 0.f);
                dd[r] = load_piece(dy, i0, N, 0.f);
            }
        }
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if ((r * G + t) * E < N)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = elem<T>(dd[r], e), xh = (elem<T>(dx_[r], e) - mean) * rstd, v = d * w[r][e];
                    a += v;                                     // past the row's end dy reads as 0, so all four sums stay
                    b = fmaf(v, xh, b);
                    sw[r][e] = fmaf(d, xh, sw[r][e]);
                    sb[r][e] += d;
                }
        const float2 c = team_sum2<G>(a, b, slot[par]);
        const float c1 = c.x * inv, c2 = c.y * inv;
        T* o = (T*)g.DX + row * g.lddx;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i0 = (r * G + t) * E;
            if (i0 < N) {
                float f[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = elem<T>(dd[r], e), xh = (elem<T>(dx_[r], e) - mean) * rstd, v = d * w[r][e];
                    f[e] = rstd * (v - fmaf(xh, c2, c1));
                }
                store_piece(o, i0, N, f);
            }
        }
    }
    float* pw = g.part + (long)blockIdx.x * 2 * N;
    if constexpr (TEAMS == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i0 = (r * G + t) * E;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i0 + e < N) { pw[i0 + e] = sw[r][e]; pw[N + i0 + e] = sb[r][e]; }
        }
    } else {
        // the workgroup's teams meet in LDS, added in team order
        __shared__ float meet[TEAMS][G * E];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < E; ++e) meet[team][t * E + e] = h ? sb[r][e] : sw[r][e];
                __syncthreads();
                for (int i = threadIdx.x; i < G * E; i += 256) {
                    float v = 0.f;
#pragma unroll
                    for (int k = 0; k < TEAMS; ++k) v += meet[k][i];
                    const int col = r * G * E + i;
                    if (col < N) pw[h * N + col] = v;
                }
            }
    }
}

// rows too long for the registers: dx with two walks over the row ...
template <class T, class WT> __global__ __launch_bounds__(1024) void ln_bwd_long_kernel(LnBwd g) {
    constexpr int E = Pack<T>::N, G = 1024;
    __shared__ float slot[2 * G / 64];
    const long row = blockIdx.x;
    const int t = threadIdx.x, N = g.N;
    const T* x = (const T*)g.X + row * g.ldx;
    const T* dy = (const T*)g.DY + row * g.lddy;
    const float mean = g.mean[row], rstd = g.rstd[row], inv = 1.f / (float)N;
    float a = 0.f, b = 0.f;
    for (long i0 = (long)t * E; i0 < N; i0 += G * E) {
        const Raw16 dx_ = load_piece(x, (int)i0, N, 0.f), dd = load_piece(dy, (int)i0, N, 0.f);
        float w[E];
        load_weights<WT, E>(w, (const WT*)g.W, (int)i0, N, 1.f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = elem<T>(dd, e) * w[e];
            a += v;
            b = fmaf(v, (elem<T>(dx_, e) - mean) * rstd, b);
        }
    }
    const float2 c = team_sum2<G>(a, b, slot);
    const float c1 = c.x * inv, c2 = c.y * inv;
    T* o = (T*)g.DX + row * g.lddx;
    for (long i0 = (long)t * E; i0 < N; i0 += G * E) {
        const Raw16 dx_ = load_piece(x, (int)i0, N, 0.f), dd = load_piece(dy, (int)i0, N, 0.f);
        float w[E], f[E];
        load_weights<WT, E>(w, (const WT*)g.W, (int)i0, N, 1.f);
#pragma unroll
        for (int e = 0; e < E; ++e)
            f[e] = rstd * (elem<T>(dd, e) * w[e] - fmaf((elem<T>(dx_, e) - mean) * rstd, c2, c1));
        store_piece(o, (int)i0, N, f);
    }
}
// ... and the column sums from a walk down the columns, one thread each, gridDim.y runs of rows
template <class T> __global__ __launch_bounds__(256) void ln_bwd_cols_kernel(LnBwd g) {
    const int col = blockIdx.x * 256 + threadIdx.x, N = g.N;
    if (col >= N) return;
    float sw = 0.f, sb = 0.f;
    for (long row = blockIdx.y; row < g.M; row += gridDim.y) {
        const float d = to_f32(((const T*)g.DY + row * g.lddy)[col]);
        sw = fmaf(d, (to_f32(((const T*)g.X + row * g.ldx)[col]) - g.mean[row]) * g.rstd[row], sw);
        sb += d;
    }
    float* pw = g.part + (long)blockIdx.y * 2 * N;
    pw[col] = sw;
    pw[N + col] = sb;
}

// dw / db = the sums of all workgroups in a fixed order: 32 columns x 32 runs of workgroups per workgroup, the runs through LDS
template <class WT>
__global__ __launch_bounds__(1024) void ln_bwd_reduce_kernel(const float* part, int blocks, int N, WT* dw, WT* db) {
    __shared__ float meet[32][33];
    const int c = threadIdx.x & 31, k = threadIdx.x >> 5;
    const long col = (long)blockIdx.x * 32 + c;                      // columns of [dw | db]
    float v = 0.f;
    if (col < 2L * N)
        for (int b = k; b < blocks; b += 32) v += part[(long)b * 2 * N + col];
    meet[k][c] = v;
    __syncthreads();
    if (k == 0 && col < 2L * N) {
        v = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) v += meet[i][c];
        if (col < N) {
            if (dw) dw[col] = from_f32<WT>(v);
        } else if (db) {
            db[col - N] = from_f32<WT>(v);
        }
    }
}

// The team of a row: the smallest whose registers hold it at R pieces per thread.
template <class T> int ln_fwd_cap(int G, int R) { return G * R * Pack<T>::N; }

template <class T, class WT> int ln_fwd(const LnFwd& g, hipStream_t st) {
    const int N = g.N, M = g.M;
#define LN_GO(G, R)                                                                                                      \
    if (N <= ln_fwd_cap<T>(G, R)) {                                                                                      \
        constexpr int TEAMS = G < 256 ? 256 / G : 1, NT = G < 256 ? 256 : G;                                             \
        hipLaunchKernelGGL((ln_fwd_kernel<T, WT, G, R>), dim3(cdiv(M, TEAMS)), dim3(NT), 0, st, g);                      \
        WFD_CHECK_LAUNCH();                                                                                              \
        return WFD_OK;                                                                                                   \
    }
    LN_GO(16, 1) LN_GO(16, 2) LN_GO(64, 1) LN_GO(64, 2) LN_GO(64, 4) LN_GO(256, 2) LN_GO(256, 4) LN_GO(1024, 2) LN_GO(1024, 4)
#undef LN_GO
    hipLaunchKernelGGL((ln_fwd_long_kernel<T, WT>), dim3(M), dim3(1024), 0, st, g);
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}

struct LnBwdShape {
    int G, R, blocks;      // R = 0: the long form
};
LnBwdShape ln_bwd_shape(int M, int N, int E) {
    const int forms[][2] = {{16, 1}, {64, 1}, {64, 2}, {256, 1}, {256, 2}, {1024, 1}, {1024, 2}};
    for (auto& f : forms)
        if (N <= f[0] * f[1] * E) {
            const int teams = f[0] < 256 ? 256 / f[0] : 1;
            const int most = f[0] == 1024 ? 256 : 512;
            const int b = cdiv(M, teams);
            return {f[0], f[1], b < most ? b : most};
        }
    return {0, 0, M < 64 ? M : 64};
}

template <class T, class WT> int ln_bwd(const LnBwd& g, WT* dw, WT* db, hipStream_t st) {
    const LnBwdShape s = ln_bwd_shape(g.M, g.N, Pack<T>::N);
    switch (s.G * 16 + s.R) {
#define LN_GO(G, R)                                                                                                      \
    case G * 16 + R:                                                                                                     \
        hipLaunchKernelGGL((ln_bwd_kernel<T, WT, G, R>), dim3(s.blocks), dim3(G < 256 ? 256 : G), 0, st, g);             \
        break;
        LN_GO(16, 1) LN_GO(64, 1) LN_GO(64, 2) LN_GO(256, 1) LN_GO(256, 2) LN_GO(1024, 1) LN_GO(1024, 2)
#undef LN_GO
        default:
            // the columns first: dx may lie over dy or x
            hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3(cdiv(g.N, 256), s.blocks), dim3(256), 0, st, g);
            hipLaunchKernelGGL((ln_bwd_long_kernel<T, WT>), dim3(g.M), dim3(1024), 0, st, g);
    }
    WFD_CHECK_LAUNCH();
    if (dw || db) {
        hipLaunchKernelGGL((ln_bwd_reduce_kernel<WT>), dim3(cdiv(2L * g.N, 32)), dim3(1024), 0, st, g.part, s.blocks, g.N, dw,
                           db);
        WFD_CHECK_LAUNCH();
    }
    return WFD_OK;
}

int elems_of(int dtype) { return dtype == WFD_F32 ? 4 : 8; }
bool rows_ok(const void* p, int ld, int M, int N, int dtype) {
    const uintptr_t align = dtype == WFD_F32 ? 3 : 1;
    return p && !((uintptr_t)p & align) && (M <= 1 || ld >= N);
}
// the longest row: 32-bit column arithmetic inside the kernels keeps 16 * 1024 elements of headroom
constexpr int LN_MAX_N = 1 << 24;

}  // namespace

extern "C" {

int wfd_layer_norm_fwd(const void* X, int ldx, int dtype, const void* weight, const void* bias, int wdtype, int M, int N,
                       float eps, void* Y, int ldy, float* mean, float* rstd, void* stream) {
    if (!wfd_dtype_ok(dtype) || (wdtype != dtype && wdtype != WFD_F32) || M < 0 || N <= 0 || N > LN_MAX_N || !(eps >= 0.f))
        return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if (!rows_ok(X, ldx, M, N, dtype) || !rows_ok(Y, ldy, M, N, dtype)) return WFD_ERR_ARG;
    LnFwd g{X, weight, bias, Y, mean, rstd, ldx, ldy, M, N, eps};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) return ln_fwd<float, float>(g, st);
    if (dtype == WFD_BF16) return wdtype == WFD_F32 ? ln_fwd<bf16_t, float>(g, st) : ln_fwd<bf16_t, bf16_t>(g, st);
    return wdtype == WFD_F32 ? ln_fwd<f16_t, float>(g, st) : ln_fwd<f16_t, f16_t>(g, st);
}

int wfd_layer_norm_bwd_floats(int M, int N, int dtype) {
    if (!wfd_dtype_ok(dtype) || M < 0 || N <= 0 || N > LN_MAX_N) return -1;
    const long n = 2L * N * ln_bwd_shape(M > 0 ? M : 1, N, elems_of(dtype)).blocks;
    return n > 0x7fffffffL ? -1 : (int)n;
}

int wfd_layer_norm_bwd(const void* DY, int lddy, const void* X, int ldx, int dtype, const void* weight, int wdtype,
                       const float* mean, const float* rstd, int M, int N, void* DX, int lddx, void* dweight, void* dbias,
                       float* part, void* stream) {
    if (!wfd_dtype_ok(dtype) || (wdtype != dtype && wdtype != WFD_F32) || M < 0 || N <= 0) return WFD_ERR_ARG;
    if (wfd_layer_norm_bwd_floats(M, N, dtype) < 0 || !part) return WFD_ERR_ARG;
    if (M > 0 && (!mean || !rstd || !rows_ok(DY, lddy, M, N, dtype) || !rows_ok(X, ldx, M, N, dtype) ||
                  !rows_ok(DX, lddx, M, N, dtype)))
        return WFD_ERR_ARG;
    LnBwd g{DY, X, weight, mean, rstd, DX, part, lddy, ldx, lddx, M, N};
    hipStream_t st = (hipStream_t)stream;
    if (M == 0) {                                        // no rows: the weights' gradients are sums of nothing
        if (wdtype == WFD_F32)
            hipLaunchKernelGGL((ln_bwd_reduce_kernel<float>), dim3(cdiv(2L * N, 32)), dim3(1024), 0, st, part, 0, N,
                               (float*)dweight, (float*)dbias);
        else                                             // a zero has the same bits in both 16-bit types
            hipLaunchKernelGGL((ln_bwd_reduce_kernel<f16_t>), dim3(cdiv(2L * N, 32)), dim3(1024), 0, st, part, 0, N,
                               (f16_t*)dweight, (f16_t*)dbias);
        WFD_CHECK_LAUNCH();
        return WFD_OK;
    }
    if (dtype == WFD_F32) return ln_bwd<float, float>(g, (float*)dweight, (float*)dbias, st);
    if (dtype == WFD_BF16)
        return wdtype == WFD_F32 ? ln_bwd<bf16_t, float>(g, (float*)dweight, (float*)dbias, st)
                                 : ln_bwd<bf16_t, bf16_t>(g, (bf16_t*)dweight, (bf16_t*)dbias, st);
    return wdtype == WFD_F32 ? ln_bwd<f16_t, float>(g, (float*)dweight, (float*)dbias, st)
                             : ln_bwd<f16_t, f16_t>(g, (f16_t*)dweight, (f16_t*)dbias, st);
}

}  // extern "C"
