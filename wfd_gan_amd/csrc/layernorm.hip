// Layer norm over the last dimension, forward and backward, fp32 / bf16 / fp16 rows with weights of the same type or fp32.
//   forward   mean = sum x / N,  rstd = 1 / sqrt(sum (x - mean)^2 / N + eps),  y = (x - mean) rstd w + b
//   backward  xh = (x - mean) rstd,  v = dy w:
//             dx = rstd (v - sum v / N - xh sum(v xh) / N),  dw = sum_rows dy xh,  db = sum_rows dy
// Bound by memory: forward reads and writes a row once, backward reads two and writes one.  A row is held packed in the registers
// of its team (16 / 64 / 256 / 1024 threads), so the variance is the two-pass one about the true mean and costs no second read.
// Measured (a large copy reaches 5.47 TB/s): forward 4096 x 2048 fp32 11.6 us = 5.8 TB/s, 8191 x 1401 bf16 10.5 us = 4.4 TB/s;
// backward 16384 x 4096 bf16 79 us = 5.1 TB/s, 5.2 of them the second launch; one row of 2048 2.1 us.  Rows beyond the registers: 2048 x
// 32768 bf16 forward 60 us = 4.5 TB/s, backward 185 = 2.2 TB/s (dx alone 105), 512 x 40001 30, 65 and 35.
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
    void* dw;          // where a single workgroup leaves them
    void* db;
    int lddy, ldx, lddx, M, N;
};

// E weights from i0 (all inside the row), `none` without weights: those are loaded all the same, from somewhere else, as in team_load
__device__ const unsigned NO_WEIGHTS[8] = {0, 0, 0, 0, 0, 0, 0, 0};
template <class WT, int E> __device__ __forceinline__ void load_weights(float* f, const WT* w, int i0, float none) {
    constexpr int P = Pack<WT>::N < E ? Pack<WT>::N : E;
    const WT* from = w ? w + i0 : (const WT*)NO_WEIGHTS;
#pragma unroll
    for (int h = 0; h < E / P; ++h) {
        const Raw16 r = load16(from + h * P);
#pragma unroll
        for (int e = 0; e < P; ++e) f[h * P + e] = w ? elem<WT>(r, e) : none;
    }
}

// those of piece `piece` of P (see team_load)
template <class WT, int E, bool ONE> __device__ __forceinline__ void team_weights(float* f, const WT* w, int piece, int P, float none) {
    if (ONE && piece >= P) return;
    load_weights<WT, E>(f, w, (ONE ? piece : min(piece, P - 1)) * E, none);
}

// ---- forward: a team of G threads per row, R pieces per thread in registers -----------------------------------------
// A team takes rows as many apart as there are teams, with the next row's loads behind it and its weights in registers: reading
// 2 N weights again for every row cost the L1's address path as much as the row itself.
template <class T, class WT, int G, int R>
__global__ __launch_bounds__(G < 256 ? 256 : G) void ln_fwd_kernel(LnFwd g) {
    constexpr int E = Pack<T>::N, TEAMS = G < 256 ? 256 / G : 1;
    constexpr bool HOLD = G < 1024 || R * E <= 16;        // a full CU of threads has 128 registers each
    __shared__ float slot[2][2][G > 64 ? G / 64 : 1];
    const int t = TEAMS > 1 ? threadIdx.x % G : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / G : 0;
    const int N = g.N, P = N / E, rest = N - P * E;       // whole pieces; the elements behind them go to the first threads
    const long step = (long)gridDim.x * TEAMS;
    long row = (long)blockIdx.x * TEAMS + team;
    if (row >= g.M) return;                               // whole teams; only teams of at most one wave share a workgroup
    const WT* W = (const WT*)g.W;
    const WT* B = (const WT*)g.B;
    // KEEP: a team of a whole CU has many empty places; those hold 0 from the start and load nothing (5000 x 10000 bf16: 51 us, reading
    // the last piece there 55; backward 75 and 82)
    constexpr bool ONE = G == 16 && R == 1, KEEP = G == 1024 && R > 1;
    Raw16 d[R];
    float last = 0.f;
    auto fetch = [&](long at) {
        const T* x = (const T*)g.X + at * g.ldx;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if constexpr (KEEP) {
                if (r * G + t < P) d[r] = load16(x + (r * G + t) * E);
            } else {
                team_load<T, ONE>(d[r], x, r * G + t, P);
            }
        if (t < rest) last = to_f32(x[P * E + t]);
    };
    if constexpr (KEEP)
#pragma unroll
        for (int r = 0; r < R; ++r) d[r] = Raw16{{0u, 0u, 0u, 0u}};
    fetch(row);
    float w[HOLD ? R : 1][E], b[HOLD ? R : 1][E], wl = 1.f, bl = 0.f;
    if constexpr (HOLD)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            team_weights<WT, E, ONE>(w[r], W, r * G + t, P, 1.f);
            team_weights<WT, E, ONE>(b[r], B, r * G + t, P, 0.f);
        }
    if (t < rest) {
        if (W) wl = to_f32(W[P * E + t]);
        if (B) bl = to_f32(B[P * E + t]);
    }
    for (int par = 0;; par ^= 1) {
        float s = last;                                   // places without an element hold 0
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (!KEEP) only(d[r], r * G + t < P, 0u);
#pragma unroll
            for (int e = 0; e < E; ++e) s += elem<T>(d[r], e);
        }
        const float mean = team_sum<G>(s, slot[par][0]) / (float)N;
        float q = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * G + t < P)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float c = elem<T>(d[r], e) - mean;
                    q = fmaf(c, c, q);
                }
        if (t < rest) q = fmaf(last - mean, last - mean, q);
        const float rstd = 1.f / sqrtf(team_sum<G>(q, slot[par][1]) / (float)N + g.eps);
        if (t == 0) {
            if (g.mean) g.mean[row] = mean;
            if (g.rstd) g.rstd[row] = rstd;
        }
        T* y = (T*)g.Y + row * g.ldy;
        const long next = row + step;
        Raw16 c[R];
#pragma unroll
        for (int r = 0; r < R; ++r) c[r] = d[r];
        const float cl = last;
        if (next < g.M) fetch(next);
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * G + t < P) {
                float o[E];
                keep_packed(c[r]);
                if constexpr (!HOLD) {
                    load_weights<WT, E>(w[0], W, (r * G + t) * E, 1.f);
                    load_weights<WT, E>(b[0], B, (r * G + t) * E, 0.f);
                }
#pragma unroll
                for (int e = 0; e < E; ++e)
                    o[e] = fmaf((elem<T>(c[r], e) - mean) * rstd, w[HOLD ? r : 0][e], b[HOLD ? r : 0][e]);
                store16(y + (r * G + t) * E, pack<T>(o));
            }
        if (t < rest) y[P * E + t] = from_f32<T>(fmaf((cl - mean) * rstd, wl, bl));
        if (next >= g.M) return;
        row = next;
    }
}

// weights i0 .. i0 + E - 1 as far as the row has them
template <class WT, int E> __device__ __forceinline__ void some_weights(float* f, const WT* w, int i0, int n, float none) {
    if (i0 + E <= n) {
        load_weights<WT, E>(f, w, i0, none);
        return;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = w && i0 + e < n ? to_f32(w[i0 + e]) : none;
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
        some_weights<WT, E>(w, (const WT*)g.W, (int)i0, N, 1.f);
        some_weights<WT, E>(b, (const WT*)g.B, (int)i0, N, 0.f);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf((elem<T>(d, e) - mean) * rstd, w[e], b[e]);
        store_piece(y, (int)i0, N, o);
    }
}

// What an element behind the last whole piece adds to the row's two sums, and its dx.  A row of one or two columns has no others, and
// there nearly everything cancels: dx of one column is 0, of two what eps leaves of the difference.  Each product is therefore rounded
// before it is added, so that equal terms cancel to the bit; fused, the one column's dx was rstd times the rounding of dy w.
__device__ __forceinline__ void rest_add(float& a, float& b, float v, float xh) {
#pragma clang fp contract(off)
    a += v;
    b += v * xh;
}
__device__ __forceinline__ float rest_dx(float rstd, float v, float xh, float c1, float c2) {
#pragma clang fp contract(off)
    return rstd * (v - c1 - xh * c2);
}
__device__ __forceinline__ float rest_product(float dy, float w) {
#pragma clang fp contract(off)
    return dy * w;
}

// ---- backward: a team walks rows, its threads keep the sums of dy xh and dy of their columns in registers ---------------
// No sum is shared while rows run, so none depends on an order; a workgroup leaves 2 N sums at its end, and a second launch adds them.
template <class T, class WT, int G, int R>
__global__ __launch_bounds__(G < 256 ? 512 : G) void ln_bwd_kernel(LnBwd g) {
    constexpr int E = Pack<T>::N, NT = G < 256 ? 512 : G, TEAMS = NT / G, W = G > 64 ? G / 64 : 1;
    constexpr bool AHEAD = R * E <= 8;                    // the next row's loads: where its registers cost no occupancy
    __shared__ float slot[2][2 * W];
    const int t = TEAMS > 1 ? threadIdx.x % G : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / G : 0;
    const int N = g.N, P = N / E, rest = N - P * E;
    constexpr bool ONE = G == 16 && R == 1, KEEP = G == 1024 && R > 1;
    float w[R][E], sw[R][E], sb[R][E], wl = 0.f, swl = 0.f, sbl = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int e = 0; e < E; ++e) { sw[r][e] = 0.f; sb[r][e] = 0.f; w[r][e] = 0.f; }
        team_weights<WT, E, ONE || KEEP>(w[r], (const WT*)g.W, r * G + t, P, 1.f);
    }
    if (t < rest) wl = g.W ? to_f32(((const WT*)g.W)[P * E + t]) : 1.f;
    const float inv = 1.f / (float)N;
    const long step = (long)gridDim.x * TEAMS;
    struct Row {
        Raw16 x[R], dy[R];
        float xl, dyl, mean, rstd;
    };
    auto fetch = [&](Row& k, long row) {
        const T* x = (const T*)g.X + row * g.ldx;
        const T* dy = (const T*)g.DY + row * g.lddy;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if constexpr (KEEP) {
                if (r * G + t < P) {
                    k.x[r] = load16(x + (r * G + t) * E);
                    k.dy[r] = load16(dy + (r * G + t) * E);
                }
            } else {
                team_load<T, ONE>(k.x[r], x, r * G + t, P);
                team_load<T, ONE>(k.dy[r], dy, r * G + t, P);
            }
        if (t < rest) { k.xl = to_f32(x[P * E + t]); k.dyl = to_f32(dy[P * E + t]); }
        k.mean = g.mean[row];
        k.rstd = g.rstd[row];
    };
    Row k;
    if constexpr (KEEP)
#pragma unroll
        for (int r = 0; r < R; ++r) k.x[r] = k.dy[r] = Raw16{{0u, 0u, 0u, 0u}};
    k.xl = k.dyl = 0.f;                                   // places without an element: dy = 0, so every sum stays
    long row = (long)blockIdx.x * TEAMS + team;
    if (row < g.M) fetch(k, row);
    for (int par = 0; row < g.M; row += step, par ^= 1) {
        Row n = k;
        if constexpr (AHEAD)
            if (row + step < g.M) fetch(n, row + step);
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (!KEEP) only(k.dy[r], r * G + t < P, 0u);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = elem<T>(k.dy[r], e), xh = (elem<T>(k.x[r], e) - k.mean) * k.rstd, v = d * w[r][e];
                a += v;
                b = fmaf(v, xh, b);
                sw[r][e] = fmaf(d, xh, sw[r][e]);
                sb[r][e] += d;
            }
        }
        const float xhl = (k.xl - k.mean) * k.rstd, vl = rest_product(k.dyl, wl);
        if (rest) {
            rest_add(a, b, vl, xhl);
            swl = fmaf(k.dyl, xhl, swl);
            sbl += k.dyl;
        }
        const float2 c = team_sum2<G>(a, b, slot[par]);
        const float c1 = c.x * inv, c2 = c.y * inv;
        T* o = (T*)g.DX + row * g.lddx;
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * G + t < P) {
                float f[E];
                keep_packed(k.dy[r]);
                keep_packed(k.x[r]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = elem<T>(k.dy[r], e), xh = (elem<T>(k.x[r], e) - k.mean) * k.rstd, v = d * w[r][e];
                    f[e] = k.rstd * (v - fmaf(xh, c2, c1));
                }
                store16(o + (r * G + t) * E, pack<T>(f));
            }
        if (t < rest) o[P * E + t] = from_f32<T>(rest_dx(k.rstd, vl, xhl, c1, c2));
        if constexpr (!AHEAD)
            if (row + step < g.M) fetch(n, row + step);
        k = n;
    }
    // the workgroup's sums: to its place in `part`, or, if it is the only one (32 rows of no whole piece), to the gradients
    float* pw = g.part + (long)blockIdx.x * 2 * N;
    auto out = [&](int h, int col, float v) {
        if (gridDim.x > 1) {
            pw[h * N + col] = v;
        } else {
            WT* to = (WT*)(h ? g.db : g.dw);
            if (to) to[col] = from_f32<WT>(v);
        }
    };
    if constexpr (TEAMS == 1) {
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r * G + t < P) {
                const int col = (r * G + t) * E;          // never alone: so few rows have a form of their own
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    store16(pw + col + e, pack<float>(sw[r] + e));
                    store16(pw + N + col + e, pack<float>(sb[r] + e));
                }
            }
        if (t < rest) { pw[P * E + t] = swl; pw[N + P * E + t] = sbl; }
    } else {
        // the teams meet in LDS, added in team order
        __shared__ __attribute__((aligned(16))) float meet[TEAMS][G * E];
#pragma unroll
        for (int r = 0; r <= R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int first = r < R ? r * G * E : P * E, count = r < R ? min(G * E, P * E - first) : rest;
                if (count <= 0) continue;                 // the same for the whole workgroup
                __syncthreads();
                if (r < R) {
#pragma unroll
                    for (int e = 0; e < E; ++e) meet[team][t * E + e] = h ? sb[r < R ? r : 0][e] : sw[r < R ? r : 0][e];
                } else if (t < rest) {
                    meet[team][t] = h ? sbl : swl;
                }
                __syncthreads();
                for (int i = threadIdx.x; i < count; i += NT) {
                    float v = 0.f;
#pragma unroll
                    for (int j = 0; j < TEAMS; ++j) v += meet[j][i];
                    out(h, first + i, v);
                }
            }
    }
}

// ---- backward of few rows: dx and the column sums in one launch ---------------------------------------------------------
// The first workgroups take 8 pieces of columns each and walk down all rows, the others take the rows: x and dy are read twice, but
// there are no partial sums and no second launch (two where dx lies over x or dy).
template <class T, class WT, int NT> __device__ __forceinline__ void bwd_columns(const LnBwd& g, int block) {
    constexpr int E = Pack<T>::N, W = NT / 64, STEP = NT / 8, U = 4;
    __shared__ float meet[W][2][8 * E];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, N = g.N;
    // the row's last piece ends where the row does: columns that it shares with the piece before are that one's
    auto column = [&](int p) { return min((block * 8 + p) * E, N - E); };
    const int col = column(t & 7);
    float sw[E], sb[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sw[e] = sb[e] = 0.f;
    if ((block * 8 + (t & 7)) * E < N)
        for (int r0 = t >> 3; r0 < g.M; r0 += U * STEP) {
            Raw16 x[U], dy[U];
            float mean[U], rstd[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const long row = r0 + j * STEP;
                x[j] = dy[j] = Raw16{{0u, 0u, 0u, 0u}};
                mean[j] = rstd[j] = 0.f;                  // a row past the last adds 0
                if (row < g.M) {
                    x[j] = load16((const T*)g.X + row * g.ldx + col);
                    dy[j] = load16((const T*)g.DY + row * g.lddy + col);
                    mean[j] = g.mean[row];
                    rstd[j] = g.rstd[row];
                }
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = elem<T>(dy[j], e);
                    sw[e] = fmaf(d, (elem<T>(x[j], e) - mean[j]) * rstd[j], sw[e]);
                    sb[e] += d;
                }
        }
    // lanes 8 apart hold the same columns
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) {
            sw[e] += __shfl_xor(sw[e], o, 64);
            sb[e] += __shfl_xor(sb[e], o, 64);
        }
    if (lane < 8)
#pragma unroll
        for (int e = 0; e < E; ++e) { meet[wave][0][lane * E + e] = sw[e]; meet[wave][1][lane * E + e] = sb[e]; }
    __syncthreads();
    const int h = t / (8 * E), c = t % (8 * E), at = column(c / E) + c % E;
    WT* to = (WT*)(h ? g.db : g.dw);
    if (h < 2 && at >= (block * 8 + c / E) * E && to) {   // never true for a piece behind the last
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) v += meet[w][h][c];
        to[at] = from_f32<WT>(v);
    }
}
template <class T, class WT, int G, int R> __device__ __forceinline__ void bwd_row(const LnBwd& g, int block) {
    constexpr int E = Pack<T>::N, TEAMS = G < 256 ? 256 / G : 1;
    __shared__ float slot[2 * (G > 64 ? G / 64 : 1)];
    const int t = TEAMS > 1 ? threadIdx.x % G : threadIdx.x;
    const int N = g.N, P = N / E, rest = N - P * E;
    const long row = (long)block * TEAMS + (TEAMS > 1 ? threadIdx.x / G : 0);
    if (row >= g.M) return;                               // whole teams, each inside a wave
    const T* x = (const T*)g.X + row * g.ldx;
    const T* dy = (const T*)g.DY + row * g.lddy;
    T* o = (T*)g.DX + row * g.lddx;
    const float mean = g.mean[row], rstd = g.rstd[row], inv = 1.f / (float)N;
    float xh[R][E], v[R][E], xhl = 0.f, vl = 0.f, a = 0.f, b = 0.f;
    Raw16 xr[R], dr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {                         // P >= 1: rows shorter than a piece do not come here
        team_load<T, false>(xr[r], x, r * G + t, P);
        team_load<T, false>(dr[r], dy, r * G + t, P);
        team_weights<WT, E, false>(v[r], (const WT*)g.W, r * G + t, P, 1.f);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        only(dr[r], r * G + t < P, 0u);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            xh[r][e] = (elem<T>(xr[r], e) - mean) * rstd;
            v[r][e] *= elem<T>(dr[r], e);
        }
    }
    if (t < rest) {
        xhl = (to_f32(x[P * E + t]) - mean) * rstd;
        vl = rest_product(to_f32(dy[P * E + t]), g.W ? to_f32(((const WT*)g.W)[P * E + t]) : 1.f);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            a += v[r][e];
            b = fmaf(v[r][e], xh[r][e], b);
        }
    rest_add(a, b, vl, xhl);
    const float2 c = team_sum2<G>(a, b, slot);
    const float c1 = c.x * inv, c2 = c.y * inv;
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (r * G + t < P) {
            float f[E];
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = rstd * (v[r][e] - fmaf(xh[r][e], c2, c1));
            store16(o + (r * G + t) * E, pack<T>(f));
        }
    if (t < rest) o[P * E + t] = from_f32<T>(rest_dx(rstd, vl, xhl, c1, c2));
}
template <class T, class WT, int G, int R>
__global__ __launch_bounds__(G < 256 ? 256 : G) void ln_bwd_few_kernel(LnBwd g, int first) {
    const int block = blockIdx.x + first, columns = cdiv_dev(g.N, 8 * Pack<T>::N);
    if (block < columns) bwd_columns<T, WT, (G < 256 ? 256 : G)>(g, block);
    else bwd_row<T, WT, G, R>(g, block - columns);
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
        some_weights<WT, E>(w, (const WT*)g.W, (int)i0, N, 1.f);
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
        some_weights<WT, E>(w, (const WT*)g.W, (int)i0, N, 1.f);
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
    if (col < 2L * N) {
        const float* p = part + (long)k * 2 * N + col;
        const long step = 64L * N;
        int b = k;
        for (; b + 7 * 32 < blocks; b += 8 * 32, p += 8 * step) {        // eight loads in flight
            float q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = p[i * step];
#pragma unroll
            for (int i = 0; i < 8; ++i) v += q[i];
        }
        for (; b < blocks; b += 32, p += step) v += *p;
    }
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

// The team of a row: the smallest whose registers hold it, from what was measured at 200 MB of rows (us; a large copy takes 37):
// 16-bit 1401 wide in 64 x 3 pieces 45.7 (64 x 4: 59.8, 256 x 1: 69.6), 2048 in 256 x 1 40.7 (64 x 4: 51.4), 8192 in 1024 x 1 43.1
// (256 x 4: 54.7); fp32 4096 in 256 x 4 39.6 (1024 x 1: 50.7).  Above 8192 (4096) columns a whole CU of threads is the only form that holds
// a row, half of its places empty at 9000; beside it stands the long form (twice as many rows, us, registers / long form: 9000 bf16 104 /
// 123, 12288 86 / 109, 16384 81 / 108; fp32 5000 77 / 101, 8192 77 / 88, 16384 79 / 106).  Workgroups: enough for 16 waves on each of
// 256 CUs, 32 where the team is small and holds little; fp32 rows of a wave or less hold so few weights that a team per row is faster
// (25000 x 1000 36.7, in 1024 workgroups 39.8; 32768 x 300 14.2, 16.1; bf16 1401 wide 44.9, 40.5).
template <class T, class WT> int ln_fwd(const LnFwd& g, hipStream_t st) {
    constexpr int E = Pack<T>::N;
#define LN_GO(G, R)                                                                                                      \
    if (g.N <= G * R * E) {                                                                                              \
        constexpr int TEAMS = G < 256 ? 256 / G : 1, NT = G < 256 ? 256 : G;                                             \
        const int all = cdiv(g.M, TEAMS);                                                                                \
        const int most = NT == 1024 ? 512 : G == 256 && R == 1 ? 2048 : E == 4 && G < 256 ? 1 << 20 : 1024;              \
        hipLaunchKernelGGL((ln_fwd_kernel<T, WT, G, R>), dim3(all < most ? all : most), dim3(NT), 0, st, g);             \
        WFD_CHECK_LAUNCH();                                                                                              \
        return WFD_OK;                                                                                                   \
    }
    LN_GO(16, 1) LN_GO(16, 2) LN_GO(64, 1) LN_GO(64, 2)
    LN_GO(64, 3)
    if constexpr (E == 4) { LN_GO(64, 4) } else { LN_GO(256, 1) }
    LN_GO(256, 2) LN_GO(256, 3)
    if constexpr (E == 4) { LN_GO(256, 4) } else { LN_GO(1024, 1) }
    LN_GO(1024, 2) LN_GO(1024, 4)
#undef LN_GO
    if (!launchable(g.M, 1024)) return WFD_ERR_ARG;
    hipLaunchKernelGGL((ln_fwd_long_kernel<T, WT>), dim3(g.M), dim3(1024), 0, st, g);
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}

struct LnBwdShape {
    int G, R, blocks;      // R = 0: the long form
    bool few;              // rows and columns in one launch, no partial sums
};
// Teams as in the forward, with fewer pieces: a column costs three registers more.  More workgroups hide more latency and cost 8 N
// bytes of partial sums each, written and read.  Measured at 200 MB of rows (us): 32768 x 1024 bf16 with 256 workgroups of 8 teams
// 43.0 (384: 52.4, 512: 47.2), 24000 x 2048 with 1024 of one team 64.2 (768: 68.0, 512: 83.6), 12000 x 4096 with 512 62.1 (768: 67.0,
// 256: 84.0), 6103 x 8192 with 256 71.5 (512: 78.2).  1401 wide: 64 x 3 pieces 66.0 (256 x 1: 92.7); 5000: 256 x 3 67.2 (1024 x 1:
// 84.9).  1024 x 2 (16-bit) and 1024 x 4 (fp32) pieces spill 4 to 16 of their 128 registers; the long form, which reads everything
// twice, is beside them still far behind (twice as many rows, us: 9000 bf16 141 / 328, 12288 130 / 283, 16384 130 / 258; fp32 16384 133 / 225).
// Few rows: a second launch costs more than a second reading.  us in one launch / two: 1024 rows x 100 bf16 9.8 / 12.9, x 1024 10.3 /
// 12.4, x 1401 13.8 / 12.8, x 4096 13.4 / 15.1, x 16384 28.4 / 40.6; 1536 x 1024 15.6 / 12.5; fp32 1024 x 2048 11.7 / 12.6, x 6000
// 22.9 / 19.6, 512 x 6000 13.6 / 13.9, x 16384 28.5 / 39.2; 512 x 3 bf16 (no whole piece) 13.7 / 13.4.  Those are calls from the host;
// replayed from a graph, where a second launch costs less, the border lies lower for narrow rows: 1024 rows x 100 bf16 8.1 / 6.4, x 512 8.3 /
// 6.6, x 1024 8.3 / 7.9, x 1401 10.5 / 10.4, x 2048 9.0 / 16.0, x 4096 11.5 / 17.4; fp32 x 100 7.9 / 6.0, x 1000 9.0 / 11.8, x 2048 9.9 / 12.1.  One
// border for all widths of a type loses up to 2 us there and 1 us at 1401 from the host.
LnBwdShape ln_bwd_shape(int M, int N, int E) {
    const int forms[][2] = {{16, 1}, {64, 1}, {64, 2}, {64, 3}, {256, 1}, {256, 2}, {256, 3}, {1024, 1}, {1024, 2}, {1024, 4}};
    for (auto& f : forms)
        if (N <= f[0] * f[1] * E && (f[1] * E <= 16 || f[1] == 3)) {
            if (N >= E && M <= (E == 8 || N <= 2048 ? 1024 : 512)) return {f[0], f[1], 1, true};
            const int teams = f[0] < 256 ? 512 / f[0] : 1;
            const int most = f[0] == 1024 || f[0] == 64 ? 256 : f[0] == 256 && f[1] == 1 ? 1024 : 512;
            const int b = cdiv(M, teams);
            return {f[0], f[1], b < most ? b : most, false};
        }
    const int most = N <= 1 << 23 ? 64 : 32;              // the scratch's size stays in 31 bits
    return {0, 0, M < most ? M : most, false};
}

template <class T, class WT> int ln_bwd(LnBwd g, WT* dw, WT* db, hipStream_t st) {
    g.dw = dw;
    g.db = db;
    const LnBwdShape s = ln_bwd_shape(g.M, g.N, Pack<T>::N);
    if (s.few) {
        const int columns = cdiv(g.N, 8 * Pack<T>::N), skip = dw || db ? 0 : columns;
        const bool over = g.DX == g.X || g.DX == g.DY;    // the columns are read before a row is written over them
        switch (s.G * 16 + s.R) {
#define LN_GO(G, R)                                                                                                      \
    case G * 16 + R: {                                                                                                   \
        const int rows = cdiv(g.M, G < 256 ? 256 / G : 1);                                                               \
        if (over && !skip)                                                                                               \
            hipLaunchKernelGGL((ln_bwd_few_kernel<T, WT, G, R>), dim3(columns), dim3(G < 256 ? 256 : G), 0, st, g, 0);   \
        hipLaunchKernelGGL((ln_bwd_few_kernel<T, WT, G, R>), dim3(rows + (over ? 0 : columns - skip)),                   \
                           dim3(G < 256 ? 256 : G), 0, st, g, over ? columns : skip);                                    \
        break;                                                                                                           \
    }
            LN_GO(16, 1) LN_GO(64, 1) LN_GO(64, 2) LN_GO(64, 3) LN_GO(256, 1) LN_GO(256, 2) LN_GO(256, 3) LN_GO(1024, 1)
            LN_GO(1024, 2)
            case 1024 * 16 + 4:
                if constexpr (sizeof(T) == 4) {           // the shape's rule gives 16-bit rows at most 2 pieces
                    if (over && !skip)
                        hipLaunchKernelGGL((ln_bwd_few_kernel<T, WT, 1024, 4>), dim3(columns), dim3(1024), 0, st, g, 0);
                    hipLaunchKernelGGL((ln_bwd_few_kernel<T, WT, 1024, 4>), dim3(g.M + (over ? 0 : columns - skip)), dim3(1024),
                                       0, st, g, over ? columns : skip);
                }
                break;
#undef LN_GO
        }
        WFD_CHECK_LAUNCH();
        return WFD_OK;
    }
    switch (s.G * 16 + s.R) {
#define LN_GO(G, R)                                                                                                      \
    case G * 16 + R:                                                                                                     \
        hipLaunchKernelGGL((ln_bwd_kernel<T, WT, G, R>), dim3(s.blocks), dim3(G < 256 ? 512 : G), 0, st, g);             \
        break;
        LN_GO(16, 1) LN_GO(64, 1) LN_GO(64, 2) LN_GO(64, 3) LN_GO(256, 1) LN_GO(256, 2) LN_GO(256, 3) LN_GO(1024, 1) LN_GO(1024, 2)
        case 1024 * 16 + 4:
            if constexpr (sizeof(T) == 4)                 // the shape's rule gives 16-bit rows at most 2 pieces
                hipLaunchKernelGGL((ln_bwd_kernel<T, WT, 1024, 4>), dim3(s.blocks), dim3(1024), 0, st, g);
            break;
#undef LN_GO
        default:
            if (!launchable(g.M, 1024)) return WFD_ERR_ARG;
            // the columns first: dx may lie over dy or x
            if (dw || db) hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3(cdiv(g.N, 256), s.blocks), dim3(256), 0, st, g);
            hipLaunchKernelGGL((ln_bwd_long_kernel<T, WT>), dim3(g.M), dim3(1024), 0, st, g);
    }
    WFD_CHECK_LAUNCH();
    if ((dw || db) && (s.G == 0 || s.blocks > 1)) {
        hipLaunchKernelGGL((ln_bwd_reduce_kernel<WT>), dim3(cdiv(2L * g.N, 32)), dim3(1024), 0, st, g.part, s.blocks, g.N, dw,
                           db);
        WFD_CHECK_LAUNCH();
    }
    return WFD_OK;
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
    if (!rows_ok(X, ldx, M, N, dtype) || !rows_ok(Y, ldy, M, N, dtype) || !same_rows(Y, ldy, X, ldx, M)) return WFD_ERR_ARG;
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
                  !rows_ok(DX, lddx, M, N, dtype) || !same_rows(DX, lddx, DY, lddy, M) || !same_rows(DX, lddx, X, ldx, M)))
        return WFD_ERR_ARG;
    LnBwd g{DY, X, weight, mean, rstd, DX, part, nullptr, nullptr, lddy, ldx, lddx, M, N};
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
