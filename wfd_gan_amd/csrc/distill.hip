// Loss of a student that learns from a teacher's K top logits (and, mixed in, from a label), with its gradient.
// Teacher: entries j with index i_j and value t_j, q = softmax(t / T) over the entries that are there (index >= 0).
// Student row x over V classes, p = softmax(x / T), p1 = softmax(x):
//   loss = w T^2 sum_j q_j (ln q_j - ln p(i_j)) - u ln p1(y)
//   d x_i = r (w T (p_i [any entry] - sum_{j: i_j = i} q_j) + u (p1_i - [i = y]))          r = grad_scale * row_scale[row]
// An index that occurs twice counts twice.  No entry (or none above -inf): the first term is 0; y < 0: the second is 0; a row without
// either has gradient 0 whatever it holds, NaN too.
// A row that holds nothing but -inf has loss +inf and gradient 0; an index or label >= V makes its row NaN.
// Bound by memory: the row is read once and, with a gradient, written once.  In between it stays packed in the registers of its
// team (up to 1024 threads x 16 pieces: 131072 16-bit or 65536 fp32 classes), so that maximum, sum and gradient cost one read.  A few
// long rows are split over workgroups instead: partial sums in a first launch, loss and gradient in a second.
// Measured (a large copy reaches 5.47 TB/s): 2048 x 128000 bf16 with gradient 210 us = 5.0 TB/s, loss alone 97 us = 5.4 TB/s; 4096 x
// 32000 bf16 105 us = 5.0 TB/s, loss alone 47 us = 5.6 TB/s; 128 x 100 fp32 5.5 us.  Split rows, read twice: 500 x 200000 bf16 with gradient
// 128 us = 3.1 TB/s, 390 x 128000 fp32 123.
#include "rowops.h"

namespace {

constexpr int MAX_ENTRIES = 256;

struct Distill {
    const void* X;
    const int* t_idx;
    const float* t_val;
    const int* labels;
    const float* row_scale;
    float* loss;
    void* DX;
    float* work;            // split form: [M][3 * splits + MAX_ENTRIES + 1]: partial sums, the entries' and the label's logits
    int ld, lddx, ldt, M, V, K;
    float temp, c, w, u, scale;     // c = log2(e) / temp
    int splits, chunk;      // split form: parts of a row, their length
    bool past;              // the gradient is written past the caches
};

__device__ __forceinline__ void wave_sync() {           // LDS traffic between the lanes of one wave
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A row's teacher entries in LDS, worked on by L lanes of one wave: where they point, exp((t - max) / T), the student's logits there.
struct Entries {
    int* at;
    float* e;
    float* x;
};
__device__ __forceinline__ Entries entries_in(float* lds, int K) { return {(int*)lds, lds + K, lds + 2 * K}; }

struct Taught {
    float max, sum;         // of the entries that are there; sum = 0: none
    bool wrong;             // an index beyond the classes
};
template <int L> __device__ __forceinline__ Taught teacher(const Distill& g, long row, int lane, const Entries& n, float c) {
    const int K = g.K;
    Taught r{-INFINITY, 0.f, false};
    float bad = 0.f;
    for (int j = lane; j < K; j += L) {
        int at = g.t_idx[row * g.ldt + j];
        const float v = g.t_val[row * g.ldt + j];
        if (at >= g.V) { bad = 1.f; at = -1; }
        n.at[j] = at;
        n.e[j] = at < 0 ? -INFINITY : v;
        r.max = fmaxf(r.max, n.e[j]);
    }
    r.max = fmaxf(lanes_max<L>(r.max), LOWEST);
    for (int j = lane; j < K; j += L) {
        n.e[j] = exp2_of((n.e[j] - r.max) * c);
        r.sum += n.e[j];
    }
    r.sum = lanes_sum<L>(r.sum);
    r.wrong = lanes_max<L>(bad) != 0.f;
    return r;
}
template <class T, int L> __device__ __forceinline__ void entries_gather(const T* x, int K, int lane, const Entries& n) {
    for (int j = lane; j < K; j += L) n.x[j] = n.at[j] >= 0 ? to_f32(x[n.at[j]]) : 0.f;
}

struct RowSums {
    float m, s, s1;         // maximum (floored), sum exp((x - m) / T), sum exp(x - m)
};

template <bool TWO> __device__ __forceinline__ void sums_to(RowSums& a, float m, float c) {      // to a maximum m >= a.m
    const float d = fmaxf(a.m - m, -1e30f);
    a.s *= exp2_of(d * c);
    if constexpr (TWO) a.s1 *= exp2_of(d * LOG2E);
    a.m = m;
}

// adds N elements whose maximum is `top`
template <bool TWO, int N> __device__ __forceinline__ void sums_add(RowSums& a, const float (&f)[N], float top, float c) {
    if (top > a.m) sums_to<TWO>(a, top, c);
    const float R = a.m * c, R1 = a.m * LOG2E;
    float s = 0.f, s1 = 0.f;
    if (fabsf(R) < WIDE && (!TWO || fabsf(R1) < WIDE)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            s += exp2_of(fmaf(f[e], c, -R));
            if constexpr (TWO) s1 += exp2_of(fmaf(f[e], LOG2E, -R1));
        }
        a.s = fmaf(exp2_of(-fmaf(a.m, c, -R)), s, a.s);
        if constexpr (TWO) a.s1 = fmaf(exp2_of(-fmaf(a.m, LOG2E, -R1)), s1, a.s1);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float z = f[e] - a.m;
            s += exp2_of(z * c);
            if constexpr (TWO) s1 += exp2_of(z * LOG2E);
        }
        a.s += s;
        if constexpr (TWO) a.s1 += s1;
    }
}

// the row's loss (every lane), from the entries and the sums
template <int L>
__device__ __forceinline__ float row_loss(const Distill& g, long row, int lane, const Entries& n, const Taught& t, const RowSums& s,
                                          int y, float xy, bool wrong) {
    // ln q_j - ln p_j = ((t_j - max t) - (x_j - max x)) / T + ln(s / sum e): terms of tens whose sum may be small, so they are added
    // in 64 bits
    const bool empty = s.s == 0.f;
    double sum = 0., apart = 0.;
    for (int j = lane; j < g.K; j += L)
        if (n.e[j] != 0.f) {
            sum += n.e[j];
            apart += n.e[j] * ((double)(g.t_val[row * g.ldt + j] - t.max) - (double)(n.x[j] - s.m));
        }
    sum = lanes_sum<L>(sum);
    apart = lanes_sum<L>(apart);
    double loss = 0.;
    if (sum != 0.) {
        const float inv = 1.f / (float)sum;
        loss = (double)g.w * g.temp * (empty ? INFINITY : (double)g.temp * logf(s.s * inv) + apart * inv);
    }
    if (y >= 0) loss -= g.u * (empty ? -INFINITY : (double)(xy - s.m) - logf(s.s1));
    return wrong ? NAN : (float)loss;
}

// what a gradient element is made of: d = cw exp((x - m) / T) + cu exp(x - m), less the targets at the entries and the label
struct GradRow {
    float m, cw, cu, r, rt;        // r = grad_scale * row_scale, rt = r w T / (sum of the teacher's exponentials)
    float R, R1, kw, ku;           // m c and m log2(e) rounded, cw and cu with what the rounding left
    bool wide;                     // m c beyond WIDE, or no term left
    bool none;                     // no term left: gradient 0
};
template <bool TWO>
__device__ __forceinline__ GradRow grad_row(const Distill& g, long row, const Taught& t, const RowSums& s, int y, bool wrong,
                                            float c) {
    GradRow d;
    d.m = s.m;
    d.r = g.scale * (g.row_scale ? g.row_scale[row] : 1.f);
    const bool empty = s.s == 0.f, on = t.sum != 0.f;
    d.rt = on ? d.r * g.w * g.temp / t.sum : 0.f;
    d.cw = on ? d.r * g.w * g.temp / s.s : 0.f;
    d.cu = y >= 0 ? d.r * g.u / s.s1 : 0.f;
    if (empty) d.cw = d.cu = 0.f;
    if (wrong) d.r = d.cw = d.cu = NAN;              // also where nothing else is left of the row
    if constexpr (!TWO) d.cw += d.cu;
    d.R = d.m * c;
    d.R1 = d.m * LOG2E;
    d.none = !on && y < 0 && !wrong;
    d.wide = d.none || !(fabsf(d.R) < WIDE && fabsf(d.R1) < WIDE);       // one test per piece for both
    d.kw = d.cw * exp2_of(-fmaf(d.m, c, -d.R));
    d.ku = d.cu * exp2_of(-fmaf(d.m, LOG2E, -d.R1));
    return d;
}
template <bool TWO> __device__ __forceinline__ float grad_dense(const GradRow& d, float x, float c) {
    if (!d.wide) {
        const float v = d.kw * exp2_of(fmaf(x, c, -d.R));
        return TWO ? fmaf(d.ku, exp2_of(fmaf(x, LOG2E, -d.R1)), v) : v;
    }
    if (d.none) return 0.f;
    const float v = d.cw * exp2_of((x - d.m) * c);
    return TWO ? fmaf(d.cu, exp2_of((x - d.m) * LOG2E), v) : v;
}
template <class T, bool TWO>
__device__ __forceinline__ void grad_piece(const GradRow& d, const Raw16& p, T* o, float c, bool past) {
    constexpr int E = Pack<T>::N;
    float f[E];
    if (!d.wide) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            f[e] = d.kw * exp2_of(fmaf(elem<T>(p, e), c, -d.R));
            if constexpr (TWO) f[e] = fmaf(d.ku, exp2_of(fmaf(elem<T>(p, e), LOG2E, -d.R1)), f[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = grad_dense<TWO>(d, elem<T>(p, e), c);
    }
    store16(o, pack<T>(f), past);
}
// the elements with a target, whole again: the first occurrence of an index subtracts all of its entries, the label its own.
// Only those of [lo, hi); runs after a barrier behind the stores that it overwrites.
template <class T, bool TWO, int L>
__device__ __forceinline__ void grad_targets(const Distill& g, const GradRow& d, const Entries& n, bool empty, int lane, T* o, int lo,
                                             int hi, int y, float xy, float c) {
    if (empty) return;
    bool label_seen = false;
    // does any index occur twice?  An entry per lane answers with scalar work; more entries are compared one by one
    bool twice = L < 64 || g.K > 64;
    if (!twice) {
        const int mine = lane < g.K ? n.at[lane] : -1;
        for (int i = 0; i < g.K && !twice; ++i) {
            const int at = __builtin_amdgcn_readlane(mine, i);
            twice = at >= 0 && __popcll(__ballot(mine == at)) > 1;
        }
    }
    for (int j = lane; j < g.K; j += L) {
        const int at = n.at[j];
        if (at < lo || at >= hi) continue;
        float sum = twice ? 0.f : n.e[j];
        bool first = true;
        if (twice)
            for (int i = 0; i < g.K; ++i)
                if (n.at[i] == at) {
                    sum += n.e[i];
                    first = first && i >= j;
                }
        if (at == y) label_seen = true;
        if (first) {
            float v = grad_dense<TWO>(d, n.x[j], c) - d.rt * sum;
            if (at == y) v -= d.r * g.u;
            o[at] = from_f32<T>(v);
        }
    }
    const bool seen = lanes_max<L>(label_seen ? 1.f : 0.f) != 0.f;
    if (lane == 0 && !seen && y >= lo && y < hi && y < g.V) o[y] = from_f32<T>(grad_dense<TWO>(d, xy, c) - d.r * g.u);
}

// ---- a row in the registers of a team of G threads ----------------------------------------------------------------------------
// TWO: a label is mixed in at a temperature other than 1, so two sums of exponentials are kept.  Without, every exponential serves both
// terms and cu joins cw.
// One row per team: the other workgroups of a CU, or of the chip where a row fills a CU's registers, keep memory busy while this one
// computes.  What matters is that all of a thread's loads are on their way before the first is waited for; walking rows with the
// next one's loads behind each stored piece was no better once that held (2048 x 128000 bf16: 205 us, walking 234; 4096 x 32000:
// 105, 105; loss alone 46, 47).
template <class T, int G, int R, bool TWO, bool GRAD>
__global__ __launch_bounds__(G < 256 ? 256 : G, R == 16 ? 4 : 1) void distill_kernel(Distill g) {
    constexpr int E = Pack<T>::N, TEAMS = G < 256 ? 256 / G : 1, L = G < 64 ? G : 64, B = R < 4 ? R : 4;
    extern __shared__ float lds[];
    __shared__ float slot[2][2 * (G > 64 ? G / 64 : 1)], told[3];
    const int t = TEAMS > 1 ? threadIdx.x % G : threadIdx.x, team = TEAMS > 1 ? threadIdx.x / G : 0, V = g.V;
    const int row = blockIdx.x * TEAMS + team;
    if (row >= g.M) return;                                   // whole teams, each inside a wave
    const float c = g.c;
    // piece r * G + t of the whole ones; the elements around them go to the first threads
    const unsigned lane_off = (unsigned)t * E;
    const T* x = (const T*)g.X + (long)row * g.ld;
    const int head = G > 64 ? off_border(x) : 0, P = (V - head) / E, rest = V - P * E;
    Raw16 d[R];
#pragma unroll
    for (int r = 0; r < R; ++r) team_load<T, G == 16 && R == 1>(d[r], x + head, r * G + t, P);
    const float tail = t < rest ? to_f32(x[t < head ? 0 : P * E + t]) : -INFINITY;
    // not always the first wave: that one sits on the same SIMD in every workgroup
    const int lane = G > 64 ? t & 63 : t;
    const bool boss = G <= 64 || (t >> 6) == (row & (G / 64 - 1));
    const Entries n = entries_in(lds + team * 3 * g.K, g.K);
    const int y = g.u != 0.f ? g.labels[row] : -1;
    const float xy = y >= 0 && y < V ? to_f32(x[y]) : 0.f;
    Taught tt{LOWEST, 0.f, false};
    if (boss) {
        tt = teacher<L>(g, row, lane, n, c);
        wave_sync();
        entries_gather<T, L>(x, g.K, lane, n);
        if constexpr (G > 64)
            if (lane == 0) { told[0] = tt.max; told[1] = tt.sum; told[2] = tt.wrong ? 1.f : 0.f; }
    }
    // per thread about its own running maximum, four pieces at a time, while later pieces are still on their way
    const unsigned none = raw_fill<T>(-INFINITY);
    RowSums s{LOWEST, 0.f, 0.f};
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += B) {
        float f[B * E], top = -INFINITY;
#pragma unroll
        for (int r = 0; r < B; ++r) {
            // every form holds at most twice the classes of the one before, so the first half of its places is full
            if (R == 1 || r0 + r >= R / 2) only(d[r0 + r], (r0 + r) * G + t < P, none);
            keep_packed(d[r0 + r]);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[r * E + e] = elem<T>(d[r0 + r], e);
                top = fmaxf(top, f[r * E + e]);
            }
        }
        sums_add<TWO>(s, f, top, c);
    }
    if (rest) {
        const float f[1] = {tail};
        sums_add<TWO>(s, f, tail, c);
    }
    sums_to<TWO>(s, team_max<G>(s.m, slot[0]), c);
    if constexpr (G > 64) tt = Taught{told[0], told[1], told[2] != 0.f};
    if constexpr (TWO) {
        const float2 q = team_sum2<G>(s.s, s.s1, slot[1]);
        s.s = q.x;
        s.s1 = q.y;
    } else {
        s.s1 = s.s = team_sum<G>(s.s, slot[1]);
    }
    const bool wrong = tt.wrong || y >= V;
    if (boss) {
        wave_sync();
        const float loss = row_loss<L>(g, row, lane, n, tt, s, y, xy, wrong);
        if (lane == 0) g.loss[row] = loss;
    }
    if constexpr (GRAD) {
        const GradRow k = grad_row<TWO>(g, row, tt, s, y, wrong, c);
        T* o = (T*)g.DX + (long)row * g.lddx;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            keep_packed(d[r]);
            if (r * G + t < P) grad_piece<T, TWO>(k, d[r], o + head + r * G * E + lane_off, c, g.past);
        }
        if (t < rest) o[t < head ? 0 : P * E + t] = from_f32<T>(grad_dense<TWO>(k, tail, c));
        if constexpr (G > 64) __syncthreads();
        else wave_sync();
        if (boss) grad_targets<T, TWO, L>(g, k, n, s.s == 0.f, lane, o, 0, V, y, xy, c);
    }
}

// ---- rows split over workgroups -------------------------------------------------------------------------------------------------
constexpr int U = 4;
template <class T, bool TWO> __global__ __launch_bounds__(256) void distill_part_kernel(Distill g) {
    constexpr int E = Pack<T>::N;
    __shared__ float slot[3][8];
    const long row = blockIdx.x / g.splits;
    const int sp = (int)(blockIdx.x - row * g.splits), t = threadIdx.x;
    const int lo = sp * g.chunk, n = min(g.chunk, g.V - lo);
    const T* x = (const T*)g.X + row * g.ld;
    float* w = g.work + row * (3L * g.splits + MAX_ENTRIES + 1);
    const float c = g.c;
    RowSums a{LOWEST, 0.f, 0.f};
    const int P = n / E, rest = n - P * E;
    const unsigned none = raw_fill<T>(-INFINITY);
    for (int p0 = 0; p0 < P; p0 += 256 * U) {
        Raw16 d[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            d[j] = Raw16{{none, none, none, none}};
            if (p0 + j * 256 + t < P) d[j] = load16(x + lo + (long)(p0 + j * 256 + t) * E);
        }
        float f[U * E], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                f[j * E + e] = elem<T>(d[j], e);
                top = fmaxf(top, f[j * E + e]);
            }
        sums_add<TWO>(a, f, top, c);
    }
    if (t < rest) {
        const float f[1] = {to_f32(x[lo + P * E + t])};
        sums_add<TWO>(a, f, f[0], c);
    }
    const float m = team_max<256>(a.m, slot[0]);
    sums_to<TWO>(a, m, c);
    const float2 q = team_sum2<256>(a.s, a.s1, slot[1]);
    if (t == 0) { w[3 * sp] = m; w[3 * sp + 1] = q.x; w[3 * sp + 2] = TWO ? q.y : q.x; }
    // the logits that the second launch needs by index, before a gradient in place could lie over them
    if (sp == 0) {
        if (t < g.K) {
            const int at = g.t_idx[row * g.ldt + t];
            w[3 * g.splits + t] = at >= 0 && at < g.V ? to_f32(x[at]) : 0.f;
        }
        if (t == 0) {
            const int y = g.u != 0.f ? g.labels[row] : -1;
            w[3 * g.splits + MAX_ENTRIES] = y >= 0 && y < g.V ? to_f32(x[y]) : 0.f;
        }
    }
}
template <class T, bool TWO> __global__ __launch_bounds__(256) void distill_finish_kernel(Distill g) {
    constexpr int E = Pack<T>::N, STEP = 256 * U * E;
    extern __shared__ float lds[];
    __shared__ float told[8];
    const int parts = g.DX ? cdiv_dev(g.V, STEP) : 1;
    const long row = blockIdx.x / parts;
    const int lo = (int)(blockIdx.x - row * parts) * STEP, t = threadIdx.x, V = g.V;
    const T* x = (const T*)g.X + row * g.ld;
    const float* w = g.work + row * (3L * g.splits + MAX_ENTRIES + 1);
    const float c = g.c;
    const Entries n = entries_in(lds, g.K);
    const int y = g.u != 0.f ? g.labels[row] : -1;
    Raw16 d[U];
    // this workgroup's whole pieces, and one of the elements behind the last of them
    const int hi = min(lo + STEP, V), P = (hi - lo) / E, rest = hi - lo - P * E;
    float tail = 0.f;
    if (g.DX) {
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (j * 256 + t < P) d[j] = load16(x + lo + (j * 256 + t) * E);
        if (t < rest) tail = to_f32(x[lo + P * E + t]);
    }
    float xy = 0.f;
    Taught tt{LOWEST, 0.f, false};
    RowSums s{LOWEST, 0.f, 0.f};
    if (t < 64) {
        // splits <= 64: a lane per part, met in a fixed order
        if (t < g.splits) s = RowSums{w[3 * t], w[3 * t + 1], w[3 * t + 2]};
        xy = w[3 * g.splits + MAX_ENTRIES];
        for (int j = t; j < g.K; j += 64) n.x[j] = w[3 * g.splits + j];
        tt = teacher<64>(g, row, t, n, c);
        sums_to<true>(s, lanes_max<64>(s.m), c);
        s.s = lanes_sum<64>(s.s);
        s.s1 = lanes_sum<64>(s.s1);
        if (t == 0) {
            told[0] = tt.max; told[1] = tt.sum; told[2] = tt.wrong ? 1.f : 0.f;
            told[3] = s.m; told[4] = s.s; told[5] = s.s1;
        }
        if (lo == 0) {
            wave_sync();
            const float loss = row_loss<64>(g, row, t, n, tt, s, y, xy, tt.wrong || y >= V);
            if (t == 0) g.loss[row] = loss;
        }
    }
    if (!g.DX) return;
    __syncthreads();
    tt = Taught{told[0], told[1], told[2] != 0.f};
    s = RowSums{told[3], told[4], told[5]};
    const GradRow k = grad_row<TWO>(g, row, tt, s, y, tt.wrong || y >= V, c);
    T* o = (T*)g.DX + row * g.lddx;
#pragma unroll
    for (int j = 0; j < U; ++j)
        if (j * 256 + t < P) grad_piece<T, TWO>(k, d[j], o + lo + (j * 256 + t) * E, c, g.past);
    if (t < rest) o[lo + P * E + t] = from_f32<T>(grad_dense<TWO>(k, tail, c));
    __syncthreads();
    if (t < 64) grad_targets<T, TWO, 64>(g, k, n, s.s == 0.f, t, o, lo, hi, y, xy, c);
}

constexpr int MAX_V = 1 << 23;

// Rows stay in registers up to 1024 threads x 16 pieces; longer ones are split, and so are the longest of these with a gradient
// where there are too few to give every CU its own (us, split and whole: 128000 bf16 classes 1 row 11.9, 16.4; 64 rows 16.1, 18.9; 96
// rows 20.6, 19.8; 66000 classes 96 rows 15.4, 16.8; 50000 classes 1 row 11.9, 11.4; loss alone of 1 x 128000 11.2, 9.3; fp32 65000
// classes 32 rows 12.6, 13.5; 64 rows 15.2, 13.9).
struct DistillShape {
    int splits, chunk;                // splits = 0: the register form
};
DistillShape distill_shape(int M, int V, int dtype, bool grad) {
    const int E = elems_of(dtype);
    if (V <= 1024 * 16 * E && (V <= 512 * 16 * E || M > (E == 8 ? 80 : 32) || !grad)) return {0, V};
    const int step = 256 * U * E, steps = cdiv(V, step);
    int S = M >= 1024 ? 1 : cdiv(1024, M > 0 ? M : 1);
    if (S > steps) S = steps;
    if (S > 64) S = 64;
    const int each = cdiv(steps, S);
    return {cdiv(steps, each), each * step};
}

template <class T, bool TWO, bool GRAD> int distill(Distill g, hipStream_t st) {
    constexpr int E = Pack<T>::N;
    const DistillShape s = distill_shape(g.M, g.V, sizeof(T) == 4 ? WFD_F32 : WFD_BF16, GRAD);
    g.splits = s.splits;
    g.chunk = s.chunk;
    if (s.splits == 0) {
#define WFD_GO(G, R)                                                                                                     \
    if (g.V <= G * R * E) {                                                                                              \
        constexpr int TEAMS = G < 256 ? 256 / G : 1;                                                                     \
        const int blocks = cdiv(g.M, TEAMS);                                                                             \
        if (!launchable(blocks, G < 256 ? 256 : G)) return WFD_ERR_ARG;                                                  \
        hipLaunchKernelGGL((distill_kernel<T, G, R, TWO, GRAD>), dim3(blocks), dim3(G < 256 ? 256 : G),                  \
                           (size_t)TEAMS * 3 * g.K * 4, st, g);                                                          \
        WFD_CHECK_LAUNCH();                                                                                              \
        return WFD_OK;                                                                                                   \
    }
        WFD_GO(16, 1) WFD_GO(16, 2) WFD_GO(64, 1) WFD_GO(64, 2) WFD_GO(64, 4) WFD_GO(64, 8) WFD_GO(256, 4) WFD_GO(256, 8) WFD_GO(256, 16)
        WFD_GO(512, 16) WFD_GO(1024, 16)
#undef WFD_GO
    }
    const int parts = g.DX ? cdiv(g.V, 256 * U * E) : 1;
    if (!launchable((long)g.M * s.splits, 256) || !launchable((long)g.M * parts, 256)) return WFD_ERR_ARG;
    hipLaunchKernelGGL((distill_part_kernel<T, TWO>), dim3(g.M * s.splits), dim3(256), 0, st, g);
    WFD_CHECK_LAUNCH();
    hipLaunchKernelGGL((distill_finish_kernel<T, TWO>), dim3(g.M * parts), dim3(256), (size_t)3 * g.K * 4, st, g);
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}
template <class T> int distill(const Distill& g, hipStream_t st) {
    if (g.temp != 1.f && g.u != 0.f) return g.DX ? distill<T, true, true>(g, st) : distill<T, true, false>(g, st);
    return g.DX ? distill<T, false, true>(g, st) : distill<T, false, false>(g, st);
}

}  // namespace

extern "C" {

int wfd_distill_floats(int M, int V, int dtype) {
    if (!wfd_dtype_ok(dtype) || M < 0 || V <= 0 || V > MAX_V) return -1;
    const DistillShape s = distill_shape(M, V, dtype, true);           // the form without a gradient never needs more
    if (M == 0 || s.splits == 0) return 0;
    const long n = (long)M * (3 * s.splits + MAX_ENTRIES + 1);
    return n > 0x7fffffffL ? -1 : (int)n;
}

int wfd_distill(const void* logits, int ldl, int dtype, int M, int V, const int* t_index, const float* t_value, int ldt, int K,
                const int* labels, float temperature, float weight, float label_weight, const float* row_scale,
                float grad_scale, float* loss, void* dlogits, int lddl, float* work, void* stream) {
    const int need = wfd_distill_floats(M, V, dtype);
    if (need < 0 || (M > 0 && need > 0 && !work) || K < 0 || K > MAX_ENTRIES || !(temperature >= 1e-6f) || !(temperature <= 1e6f))
        return WFD_ERR_ARG;
    if (!(weight - weight == 0.f) || !(label_weight - label_weight == 0.f)) return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if (label_weight != 0.f && !labels) return WFD_ERR_ARG;
    if (!loss || !rows_ok(logits, ldl, M, V, dtype) || (dlogits && !rows_ok(dlogits, lddl, M, V, dtype))) return WFD_ERR_ARG;
    if (!same_rows(dlogits, lddl, logits, ldl, M)) return WFD_ERR_ARG;
    if (K > 0 && (!t_index || !t_value || (M > 1 && ldt < K))) return WFD_ERR_ARG;
    // without weight the entries are not read, and the label's term has no temperature
    if (weight == 0.f) K = 0;
    if (K == 0) temperature = 1.f;
    Distill g{logits, t_index, t_value, labels, row_scale, loss, dlogits, work, ldl, lddl, ldt, M, V, K, temperature,
              log2e_over(temperature), weight, label_weight, grad_scale, 0, 0, past_caches(M, V, dtype == WFD_F32 ? 4 : 2)};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) return distill<float>(g, st);
    return dtype == WFD_BF16 ? distill<bf16_t>(g, st) : distill<f16_t>(g, st);
}

}  // extern "C"
