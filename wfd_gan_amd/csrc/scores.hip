// Scores of given labels over V classes: log probability, entropy and the k best alternatives of each row of logits, and the
// gradient of log probability and entropy.  With temperature T, m = max x, z = (x - m) / T, s = sum exp z:
//   logprob(y) = z_y - ln s,   H = ln s - (sum z exp z) / s,   p = exp z / s
//   d x_i = (1 / T) (g ([i = y] - p_i) - h p_i (ln p_i + H))
// Sums are fp32 about the row's own maximum; (m, ln s) stay apart in `stat`, so that differences to the maximum are exact.
// Bound by memory: the forward reads a row once and writes a few words, the gradient reads and writes it once.  So one walk does all:
// running maximum and sums, one exponential and four other operations per class, and for the alternatives no more than one maximum per
// 4 pieces; the few groups that can hold an alternative are read again from the caches.
// Measured (a large copy reaches 5.47 TB/s): 4096 x 50257 bf16, three buffers in turn, 84 us = 4.9 TB/s without alternatives, 95 with 10,
// 115 with 64 (one buffer again and again, part of which stays in the last-level cache: 88 with 10); the gradient of 4096 x 32000 bf16
// 94 us = 5.6 TB/s; one row of 131072 with 20 alternatives 7.2 us and 4.3 for the join.
// A row that holds nothing but -inf: logprob -inf, entropy 0, gradient 0.  NaN and +inf make the row's numbers NaN.
#include "rowops.h"

namespace {

struct Scores {
    const void* X;
    const int* labels;
    float* logprob;
    float* entropy;
    float* stat;
    float* top_lp;
    int* top_idx;
    float* work;          // [M][splits][3 + 2 k]: a part's statistics, its alternatives' values and indices
    int ld, M, V, k;
    float inv_t, c;       // 1 / T and log2(e) / T
    int splits, chunk;    // parts of a row and their length (a multiple of a step)
};
struct ScoresBwd {
    const void* X;
    const int* labels;
    const float* stat;
    const float* entropy;
    const float* d_lp;
    const float* d_ent;
    void* DX;
    int ld, lddx, M, V;
    float inv_t;
    int chunks;           // workgroups (long rows) or pieces (short rows) per row
    bool past;            // the gradient is written past the caches
};

// order of alternatives: larger value first (NaN before every number, -0 as 0), then the lower index.  NaN's place is one below the
// largest, so that the key of ~0 belongs to no element: a walk that takes one after another starts above it.
constexpr unsigned NAN_BITS = 0xfffffffeu;
__device__ __forceinline__ unsigned order_bits(float v) {
    if (v != v) return NAN_BITS;
    const unsigned u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float v, int i) {
    return ((unsigned long long)order_bits(v) << 32) | (unsigned)~i;
}

__device__ __forceinline__ float order_value(unsigned b) {
    return b == NAN_BITS ? NAN : __uint_as_float((b & 0x80000000u) ? b ^ 0x80000000u : ~b);
}

// ---- what one workgroup knows of its part of a row -----------------------------------------------------------------------
// Running statistics: m = max(largest so far, -FLT_MAX), s = sum exp2((x - m) c), u = sum exp2((x - m) c) (x - m) c with
// c = log2(e) / T.  The floor under m keeps x - m defined for rows of -inf (their s stays 0, which is how they are told) and for
// rows at the type's lowest value (x - m = 0).  exp2 of -inf is 0, and u takes no exponent below FAINT, so masked classes add
// nothing; NaN and +inf reach s as NaN.
struct Stat {
    float m, s, u;
};
__device__ __forceinline__ void stat_to(Stat& a, float m, float c) {          // moves a to a maximum m >= a.m
    const float d = fmaxf((a.m - m) * c, FAINT), w = exp2_of(d);         // floored last: s * d stays finite where w is 0
    a.u = w * fmaf(a.s, d, a.u);
    a.s *= w;
    a.m = m;
}
template <int N> __device__ __forceinline__ void stat_add(Stat& a, const float (&f)[N], float top, float c) {
    if (top > a.m) stat_to(a, top, c);
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float d = (f[e] - a.m) * c, w = exp2_of(d);     // the difference first: a lone class has s = 1 to the bit
        s += w;
        u = fmaf(w, fmaxf(d, FAINT), u);
    }
    a.u += u;
    a.s += s;
}
// over a team of G threads; slot: 3 * G / 64 floats of LDS.  Every thread gets the sum, added in a fixed order.
template <int G> __device__ __forceinline__ Stat stat_team(Stat a, float c, float* slot) {
    const float m = lanes_max<(G < 64 ? G : 64)>(a.m);
    stat_to(a, m, c);
    a.s = lanes_sum<(G < 64 ? G : 64)>(a.s);
    a.u = lanes_sum<(G < 64 ? G : 64)>(a.u);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) { slot[3 * w] = a.m; slot[3 * w + 1] = a.s; slot[3 * w + 2] = a.u; }
        __syncthreads();
        float top = slot[0];
#pragma unroll
        for (int i = 1; i < W; ++i) top = fmaxf(top, slot[3 * i]);
        Stat r{top, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < W; ++i) {
            Stat b{slot[3 * i], slot[3 * i + 1], slot[3 * i + 2]};
            stat_to(b, top, c);
            r.s += b.s;
            r.u += b.u;
        }
        a = r;
    }
    return a;
}

// what the statistics of a whole row say; `empty`: nothing but -inf
struct RowEnd {
    float m, log_s, entropy;
    bool empty;
};
__device__ __forceinline__ RowEnd row_end(const Stat& a) {
    RowEnd r;
    r.empty = a.s == 0.f;
    r.m = r.empty ? -INFINITY : a.m;
    r.log_s = r.empty ? 0.f : logf(a.s);
    r.entropy = r.empty ? 0.f : fmaf(-LN2, a.u / a.s, r.log_s);
    return r;
}
__device__ __forceinline__ float row_lp(const RowEnd& r, float x, float inv_t) {
    return r.empty ? -INFINITY : (x - r.m) * inv_t - r.log_s;
}
__device__ __forceinline__ void row_store(const Scores& g, long row, const RowEnd& r, float xy, int y) {
    if (g.stat) { g.stat[2 * row] = r.m; g.stat[2 * row + 1] = r.log_s; }
    if (g.entropy) g.entropy[row] = r.entropy;
    if (g.logprob) g.logprob[row] = y < 0 ? 0.f : y >= g.V ? NAN : row_lp(r, xy, g.inv_t);
}

// ---- alternatives of a part of a row --------------------------------------------------------------------------------------
// Every thread has left the largest value of each group of pieces that it visited in LDS.  The (k / waves)-th largest thread maximum
// of a wave (alone in its workgroup, a wave counts each thread's two largest), the smallest such of all waves, is a value that at
// least k elements reach; so is any wave's k-th largest (a part may be so short that the last waves have none).  The larger of the
// two is tau.  Only groups whose maximum reaches tau are read again, an element per thread; what reaches tau there goes to a list
// (expected length: k and a few), whose order is found by counting.  When more than the lists hold reach tau, they are ties at tau but
// for a few: those above tau are listed and the rest is filled up by walking the ties in index order.  Where that list runs over as
// well (sorted rows: thousands above tau), tau becomes the k-th largest value itself, found by counting (4096 sorted rows of 50257
// bf16, top 64: 0.54 ms, one after another 12.6).  Rows with NaN take the k largest one after another.
constexpr int U = 4;                      // pieces per group

template <int NT> struct PickLds {
    static constexpr int CAND = 4 * NT, GROUPS = 2 * NT;
    unsigned long long key[CAND];
    unsigned long long best[NT / 64 ? NT / 64 : 1];
    float tau[NT / 64 ? NT / 64 : 1], own[NT / 64 ? NT / 64 : 1];
    int group[GROUPS];
    int groups, count, run[NT / 64 ? NT / 64 : 1];
};

struct NoLds {};
template <bool PICK, int NT> struct Cond { typedef PickLds<NT> type; };
template <int NT> struct Cond<false, NT> { typedef NoLds type; };

template <int NT> __device__ __forceinline__ void team_sync() {
    if constexpr (NT > 64) __syncthreads();
    else __builtin_amdgcn_wave_barrier(), __threadfence_block();
}
template <int NT> __device__ __forceinline__ unsigned long long team_max_key(unsigned long long v, unsigned long long* slot) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    if constexpr (NT > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = slot[0];
        for (int i = 1; i < NT / 64; ++i) v = slot[i] > v ? slot[i] : v;
    }
    return v;
}

// the n-th largest (1 <= n <= 64) of the lanes' values (no NaN): a lane's value divides the lanes that are still in question, the
// masks and counts are scalar work
template <class V> __device__ __forceinline__ V lanes_nth(V v, int n) {
    unsigned long long in = ~0ull;
    for (;;) {
        const int src = __ffsll((long long)in) - 1;
        const V p = __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), src));
        const unsigned long long gt = __ballot(v > p) & in, eq = __ballot(v == p) & in;
        const int above = __popcll(gt), same = __popcll(eq);
        if (n <= above) {
            in = gt;
        } else if (n <= above + same) {
            return p;
        } else {
            n -= above + same;
            in &= ~(gt | eq);
        }
    }
}
// the n-th largest (1 <= n <= 128) of two values per lane
__device__ __forceinline__ float lanes_nth2(float a, float b, int n) {
    unsigned long long in_a = ~0ull, in_b = ~0ull;
    for (;;) {
        const float v = in_a ? a : b;
        const int src = __ffsll((long long)(in_a ? in_a : in_b)) - 1;
        const float p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), src));
        const unsigned long long gt_a = __ballot(a > p) & in_a, gt_b = __ballot(b > p) & in_b;
        const unsigned long long eq_a = __ballot(a == p) & in_a, eq_b = __ballot(b == p) & in_b;
        const int above = __popcll(gt_a) + __popcll(gt_b), same = __popcll(eq_a) + __popcll(eq_b);
        if (n <= above) {
            in_a = gt_a;
            in_b = gt_b;
        } else if (n <= above + same) {
            return p;
        } else {
            n -= above + same;
            in_a &= ~(gt_a | eq_a);
            in_b &= ~(gt_b | eq_b);
        }
    }
}

// Which of 256 bins, from the highest, holds the need-th element (need comes back as the rank inside it).  Every wave finds it.
__device__ __forceinline__ int bin_of(const int* hist, int lane, int& need) {
    int c[4], s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) s += c[i] = hist[255 - 4 * lane - i];
    int upto = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(upto, o, 64);
        if (lane >= o) upto += v;
    }
    int left = need - (upto - s), at = 0;
    const int src = (__ffsll((long long)__ballot(upto >= need)) - 1) & 63;      // at least `need` elements are counted
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (at == i && left > c[i]) { left -= c[i]; ++at; }
    need = __builtin_amdgcn_readlane(left, src);
    return 255 - 4 * src - __builtin_amdgcn_readlane(at, src);
}
// The k-th largest value of x[0, n), of which at least k reach `tau` (no NaN): four counts of eight bits of the order each.  Every count
// is a walk over the part from the caches: for rows whose large values stand together (sorted ones), where the lists run over.
template <class T, int NT> __device__ __forceinline__ float kth_value(const T* x, int n, float tau, int k, PickLds<NT>& l) {
    constexpr int E = Pack<T>::N;
    const int t = threadIdx.x, lane = t & 63;
    int* hist = (int*)l.key;
    unsigned prefix = 0;
    int need = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = t; i < 256; i += NT) hist[i] = 0;
        team_sync<NT>();
        for (long i0 = (long)t * E; i0 < n; i0 += NT * E) {
            const Raw16 d = load_piece(x, (int)i0, n, -INFINITY);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float f = elem<T>(d, e);
                const unsigned b = order_bits(f);
                if (f >= tau && i0 + e < n && (shift == 24 || b >> (shift + 8) == prefix >> (shift + 8)))
                    atomicAdd(&hist[b >> shift & 255], 1);
            }
        }
        team_sync<NT>();
        prefix |= (unsigned)bin_of(hist, lane, need) << shift;
        team_sync<NT>();
    }
    return order_value(prefix);
}

// Leaves the k best of x[0, n) (indices from `base`) at out_val / out_idx in order, places without an element as index -1.
// gmax[it * NT + t]: the group maxima of x[head, n); head (0 or 1) elements in front are in no group.  sum: the part's s (NaN tells
// of NaN or +inf).
template <class T, int NT>
__device__ __forceinline__ void pick(const T* x0, int n0, int base0, int head, int k, int niter, const float* gmax, float tmax,
                                     float next, float sum, PickLds<NT>& l, float* out_val, int* out_idx) {
    constexpr int E = Pack<T>::N, W = NT / 64, CAND = PickLds<NT>::CAND, GROUPS = PickLds<NT>::GROUPS;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const T* x = x0 + head;
    const int n = n0 - head, base = base0 + head;
    const float front = head ? to_f32(x0[0]) : 0.f;
    if (sum == sum) {
        const float share = W == 1 ? lanes_nth2(tmax, next, k) : lanes_nth(tmax, (k + W - 1) / W);
        const float own = W > 1 && n < NT * E ? lanes_nth(tmax, k) : -INFINITY;
        if (lane == 0) { l.tau[wave] = share; l.own[wave] = own; }
        if (t == 0) l.count = l.groups = 0;
        team_sync<NT>();
        float tau = l.tau[0], best = l.own[0];
#pragma unroll
        for (int i = 1; i < W; ++i) {
            tau = fminf(tau, l.tau[i]);
            best = fmaxf(best, l.own[i]);
        }
        tau = fmaxf(tau, best);
        int total = 0;
        bool ties = false;
        for (int pass = 0;; ++pass) {
            for (int it = 0; it < niter; ++it) {
                const float gm = gmax[it * NT + t];
                if (pass ? gm > tau : gm >= tau) {
                    const int at = atomicAdd(&l.groups, 1);
                    if (at < GROUPS) l.group[at] = it * NT + t;
                }
            }
            if (head && t == 0 && (pass ? front > tau : front >= tau)) {
                const int at = atomicAdd(&l.count, 1);
                if (at < CAND) l.key[at] = order_key(front, base0);
            }
            team_sync<NT>();
            const int groups = l.groups;
            // an element per thread, so that the few groups keep all lanes busy
            if (groups <= GROUPS)
                for (int a = t; a < groups * U * E; a += NT) {
                    const int id = l.group[a / (U * E)], j = a / E % U, e = a % E;
                    const int i = ((id / NT * U + j) * NT + id % NT) * E + e;
                    if (i >= n) continue;
                    const float f = to_f32(x[i]);
                    if (pass ? f > tau : f >= tau) {
                        const int at = atomicAdd(&l.count, 1);
                        if (at < CAND) l.key[at] = order_key(f, base + i);
                    }
                }
            team_sync<NT>();
            total = l.count;
            team_sync<NT>();
            if ((groups <= GROUPS && total <= CAND) || pass == 2) break;
            // fewer than k elements are above the k-th largest value, so that the third pass is the last
            if (pass == 1) tau = kth_value<T, NT>(x0, n0, tau, k, l);
            ties = true;
            if (t == 0) l.count = l.groups = 0;
            team_sync<NT>();
        }
        // order by counting: the list is short, every thread reads all of it (broadcasts)
        for (int a = t; a < total; a += NT) {
            const unsigned long long key = l.key[a];
            int rank = 0;
#pragma unroll 8
            for (int b = 0; b < total; ++b) rank += l.key[b] > key;
            if (rank < k) {
                const int i = (int)~(unsigned)key;
                out_val[rank] = to_f32(x0[i - base0]);
                out_idx[rank] = i;
            }
        }
        int have = total;
        if (ties && have < k) {
            // ties at tau in index order, E elements per thread at a time, until there are enough
            if (head && front == tau) {
                if (t == 0) { out_val[have] = tau; out_idx[have] = base0; }
                ++have;
            }
            for (long p0 = 0; p0 * E < n && have < k; p0 += NT) {
                const long i0 = (p0 + t) * E;
                unsigned hit = 0;
                if (i0 < n) {
                    const Raw16 d = load_piece(x, (int)i0, n, -INFINITY);
#pragma unroll
                    for (int e = 0; e < E; ++e) hit |= (elem<T>(d, e) == tau && i0 + e < n) ? 1u << e : 0u;
                }
                int before = __popc(hit);                           // inclusive count over the lanes
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int v = __shfl_up(before, o, 64);
                    if (lane >= o) before += v;
                }
                if (lane == 63) l.run[wave] = before;
                team_sync<NT>();
                int at = have + before - __popc(hit), all = 0;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    if (i < wave) at += l.run[i];
                    all += l.run[i];
                }
                for (int e = 0; e < E; ++e)
                    if (hit >> e & 1) {
                        if (at < k) { out_val[at] = tau; out_idx[at] = base + (int)i0 + e; }
                        ++at;
                    }
                have += all;
                team_sync<NT>();
            }
        }
        for (int a = have + t; a < k; a += NT) { out_val[a] = -INFINITY; out_idx[a] = -1; }
        return;
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < k; ++j) {
        unsigned long long best = 0;
        for (int i = t; i < n0; i += NT) {
            const unsigned long long key = order_key(to_f32(x0[i]), base0 + i);
            if (key < last && key > best) best = key;
        }
        last = team_max_key<NT>(best, l.best);
        if (t == 0) {
            const int i = (int)~(unsigned)last;
            out_val[j] = last ? to_f32(x0[i - base0]) : -INFINITY;
            out_idx[j] = last ? i : -1;
        }
    }
}

// ---- one walk over a part of a row ----------------------------------------------------------------------------------------
template <class T, int NT, bool PICK>
__device__ __forceinline__ Stat walk(const T* x, int n, float c, float* gmax, float& tmax, float& next) {
    constexpr int E = Pack<T>::N, STEP = NT * U * E;
    const int t = threadIdx.x;
    Stat a{LOWEST, 0.f, 0.f};
    tmax = next = -INFINITY;                                  // the thread's two largest group maxima
    int it = 0;
    auto take = [&](const Raw16 (&d)[U]) {
        float f[U * E];
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) f[j * E + e] = elem<T>(d[j], e);
        float top = f[0];
#pragma unroll
        for (int e = 1; e < U * E; ++e) top = fmaxf(top, f[e]);
        if constexpr (PICK) {
            gmax[it * NT + t] = top;
            if constexpr (NT == 64) next = fmaxf(next, fminf(tmax, top));
            tmax = fmaxf(tmax, top);
        }
        stat_add(a, f, top, c);
    };
    for (; (long)(it + 1) * STEP <= n; ++it) {
        Raw16 d[U];
#pragma unroll
        for (int j = 0; j < U; ++j) d[j] = load16(x + (long)it * STEP + (j * NT + t) * E);
        take(d);
    }
    if ((long)it * STEP < n) {
        // the rest, as far as any lane of the wave has a piece.  All loads first, and none under a condition (see team_load): a piece
        // that would reach past the end starts earlier, its elements before i0 are another piece's
        float group = -INFINITY;
        const int first = (t & ~63) * E, i0 = it * STEP + t * E, last = max(n - E, 0);
        Raw16 d[U];
        if (n >= E) {
#pragma unroll
            for (int j = 0; j < U; ++j) d[j] = load16(x + min(i0 + j * NT * E, last));
        } else {
            d[0] = load_piece(x, 0, n, -INFINITY);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = i0 + j * NT * E, s = min(i, last);
            if (it * STEP + j * NT * E + first >= n) continue;
            float f[E], top = -INFINITY;
            if (i < n) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    f[e] = s + e >= i ? elem<T>(d[j], e) : -INFINITY;
                    top = fmaxf(top, f[e]);
                }
                stat_add(a, f, top, c);
                group = fmaxf(group, top);
            }
        }
        if constexpr (PICK) {
            gmax[it * NT + t] = group;
            if constexpr (NT == 64) next = fmaxf(next, fminf(tmax, group));
            tmax = fmaxf(tmax, group);
        }
    }
    return a;
}

template <class T, int NT, bool PICK> __global__ __launch_bounds__(NT) void scores_kernel(Scores g) {
    constexpr int E = Pack<T>::N, STEP = NT * U * E;
    extern __shared__ float gmax[];
    __shared__ float slot[3 * (NT / 64)];
    __shared__ typename Cond<PICK, NT>::type l;
    const long part = blockIdx.x, row = part / g.splits;
    const int sp = (int)(part - row * g.splits);
    const int lo = sp * g.chunk, n = min(g.chunk, g.V - lo);
    const T* x = (const T*)g.X + row * g.ld + lo;
    const int y = g.labels ? g.labels[row] : -1;
    const float xy = g.splits == 1 && y >= 0 && y < g.V ? to_f32(x[y]) : 0.f;
    const float c = g.c;
    float tmax, next;
    const int head = off_border(x);
    Stat a = walk<T, NT, PICK>(x + head, n - head, c, gmax, tmax, next);
    if (head && threadIdx.x == 0) {
        const float f[1] = {to_f32(x[0])};
        stat_add(a, f, f[0], c);
    }
    a = stat_team<NT>(a, c, slot);
    float* w = g.work + part * (3 + 2 * g.k);
    const bool whole = g.splits == 1;
    RowEnd r{};
    if (whole) {
        r = row_end(a);
        if (threadIdx.x == 0) row_store(g, row, r, xy, y);
    } else if (threadIdx.x == 0) {
        w[0] = a.m; w[1] = a.s; w[2] = a.u;
    }
    if constexpr (PICK) {
        float* val = whole ? g.top_lp + row * g.k : w + 3;
        int* idx = whole ? g.top_idx + row * g.k : (int*)(w + 3 + g.k);
        pick<T, NT>(x, n, lo, head, g.k, cdiv_dev(n - head, STEP), gmax, tmax, next, a.s, l, val, idx);
        if (whole) {
            team_sync<NT>();
            for (int j = threadIdx.x; j < g.k; j += NT) val[j] = row_lp(r, val[j], g.inv_t);
        }
    }
}

// the parts of a row: a lane per part for the statistics, alternatives from the parts' lists
template <class T> __global__ __launch_bounds__(256) void scores_join_kernel(Scores g) {
    extern __shared__ unsigned long long keys[];              // splits * k
    constexpr int CAND = 1024;
    __shared__ unsigned long long list[CAND];
    __shared__ int count;
    const long row = blockIdx.x;
    const int t = threadIdx.x, S = g.splits, k = g.k, each = 3 + 2 * k;
    const float* w = g.work + row * S * each;
    if (t == 0) count = 0;
    const int lane = t & 63;
    // If n parts have a j-th entry that reaches a value, n j elements do: the ceil(k / j)-th largest of the parts' j-th entries, with
    // about half of the parts in it.  A lane per part (at most 64); a place without an entry counts as 0, below every number.
    const int j = min(k, cdiv_dev(2 * k, S));
    unsigned jth = 0;
    if (k > 0 && lane < S) {
        const float* p = w + lane * each + 3;
        if (((const int*)p)[k + j - 1] >= 0) jth = order_bits(p[j - 1]);
    }
    for (int i = t; i < S * k; i += 256) {
        const int s = i / k, e = i - s * k;
        const float* p = w + s * each + 3;
        const float v = p[e];
        const int at = ((const int*)p)[k + e];
        keys[i] = at < 0 ? 0ull : order_key(v, at);
    }
    const float c = g.c;
    Stat a{LOWEST, 0.f, 0.f};
    if (lane < S) a = Stat{w[lane * each], w[lane * each + 1], w[lane * each + 2]};      // S <= 64
    const RowEnd r = row_end(stat_team<64>(a, c, nullptr));
    if (t == 255) {
        const int y = g.labels ? g.labels[row] : -1;
        row_store(g, row, r, y >= 0 && y < g.V ? to_f32(((const T*)g.X + row * g.ld)[y]) : 0.f, y);
    }
    if (k == 0) return;
    const unsigned least = lanes_nth(jth, cdiv_dev(k, j));
    __syncthreads();
    for (int i = t; i < S * k; i += 256) {
        const unsigned long long key = keys[i];
        if ((unsigned)(key >> 32) >= least && key) {
            const int at = atomicAdd(&count, 1);
            if (at < CAND) list[at] = key;
        }
    }
    __syncthreads();
    const bool all = count > CAND;
    const unsigned long long* from = all ? keys : list;
    const int n = all ? S * k : count;
    for (int i = t; i < n; i += 256) {
        const unsigned long long key = from[i];
        if (!key) continue;
        int rank = 0;
#pragma unroll 8
        for (int b = 0; b < n; ++b) rank += from[b] > key;
        if (rank < k) {
            g.top_idx[row * k + rank] = (int)~(unsigned)key;
            g.top_lp[row * k + rank] = row_lp(r, order_value((unsigned)(key >> 32)), g.inv_t);
        }
    }
}

// ---- few classes: a team of G lanes holds the row, R pieces per lane and at most one element behind the last whole piece --------
template <int G> __device__ __forceinline__ unsigned lanes_max_u32(unsigned v) {
    auto step = [&](unsigned w) { v = w > v ? w : v; };
    step(__builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true));
    step(__builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true));
    if constexpr (G >= 32) step(__shfl_xor(v, 16, 64));
    if constexpr (G >= 64) step(__shfl_xor(v, 32, 64));
    return v;
}
constexpr int LIST = 192;                 // candidates of a wave's row
template <class T, int G, int R> __global__ __launch_bounds__(256) void scores_few_kernel(Scores g) {
    constexpr int E = Pack<T>::N, TEAMS = 256 / G, N = R * E + 1;
    __shared__ unsigned long long lists[G == 64 ? 4 : 1][G == 64 ? LIST : 1];
    const int t = threadIdx.x % G, V = g.V, P = V / E, rest = V - P * E;
    const long row = (long)blockIdx.x * TEAMS + threadIdx.x / G;
    if (row >= g.M) return;                                   // whole teams
    const T* x = (const T*)g.X + row * g.ld;
    float f[N];
    auto have = [&](int e) { return e < R * E ? (e / E) * G + t < P : t < rest; };
    auto index = [&](int e) { return e < R * E ? ((e / E) * G + t) * E + e % E : P * E + t; };
    {
        Raw16 d[R];
        const unsigned none = raw_fill<T>(-INFINITY);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            d[r] = Raw16{{none, none, none, none}};
            if (r * G + t < P) d[r] = load16(x + (r * G + t) * E);
        }
        f[R * E] = t < rest ? to_f32(x[P * E + t]) : -INFINITY;
#pragma unroll
        for (int e = 0; e < R * E; ++e) f[e] = elem<T>(d[e / E], e % E);
    }
    const int y = g.labels ? g.labels[row] : -1;
    const float xy = y >= 0 && y < V ? to_f32(x[y]) : 0.f;
    const float c = g.c;
    // the lane's two largest; a NaN is in neither, and in every sum
    float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        b2 = fmaxf(b2, fminf(b1, f[e]));
        b1 = fmaxf(b1, f[e]);
    }
    Stat a{LOWEST, 0.f, 0.f};
    stat_add(a, f, fmaxf(lanes_max<G>(b1), LOWEST), c);
    a.s = lanes_sum<G>(a.s);
    a.u = lanes_sum<G>(a.u);
    const RowEnd r = row_end(a);
    if (t == 0) row_store(g, row, r, xy, y);
    if (g.k == 0) return;
    if constexpr (G == 64) {
        // as in pick(): a value that k elements reach, a list of what reaches it, its order by counting
        if (a.s == a.s) {
            unsigned long long* list = lists[threadIdx.x >> 6];
            const float tau = lanes_nth2(b1, b2, g.k);
            const unsigned long long below = (1ull << t) - 1;
            int n = 0;
            auto gather = [&](bool strict) {
                n = 0;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const bool hit = (strict ? f[e] > tau : f[e] >= tau) && have(e);
                    const unsigned long long who = __ballot(hit);
                    if (who == 0) continue;
                    const int at = n + __popcll(who & below);
                    if (hit && at < LIST) list[at] = order_key(f[e], index(e));
                    n += __popcll(who);
                }
            };
            gather(false);
            const bool ties = n > LIST;
            if (ties) gather(true);
            if (n <= LIST) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                for (int i = t; i < n; i += 64) {
                    const unsigned long long key = list[i];
                    int rank = 0;
#pragma unroll 8
                    for (int b = 0; b < n; ++b) rank += list[b] > key;
                    if (rank < g.k) {
                        g.top_idx[row * g.k + rank] = (int)~(unsigned)key;
                        g.top_lp[row * g.k + rank] = row_lp(r, order_value((unsigned)(key >> 32)), g.inv_t);
                    }
                }
                // what is left are ties at tau, in the order of their indices: by piece, lane and element
                if (ties)
#pragma unroll
                    for (int r0 = 0; r0 <= R; ++r0) {
                        if (n >= g.k) continue;
                        unsigned long long who[E];
                        int before = 0, all = 0;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            who[e] = 0;
                            if (r0 == R && e > 0) continue;
                            who[e] = __ballot(f[r0 * E + e] == tau && have(r0 * E + e));
                            before += __popcll(who[e] & below);
                            all += __popcll(who[e]);
                        }
                        int at = n + before;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            if (r0 == R && e > 0) continue;
                            if (who[e] >> t & 1) {
                                if (at < g.k) {
                                    g.top_idx[row * g.k + at] = index(r0 * E + e);
                                    g.top_lp[row * g.k + at] = row_lp(r, tau, g.inv_t);
                                }
                                ++at;
                            }
                        }
                        n += all;
                    }
                return;
            }
        }
    }
    // one alternative after another: best of the lane, best of the team, and the winner looks for its next.  Rows with NaN, short teams,
    // and rows whose list runs over without ties (16384 sorted rows of 1500 bf16, top 64: 0.4 ms; the count of kth_value here costs
    // every row 65 registers, and random ones 50 us instead of 31)
    unsigned long long done = 0;                              // elements of this lane already given
    for (int j = 0; j < g.k; ++j) {
        unsigned best = 0;
        int at = 0x7fffffff, slot = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const unsigned b = order_bits(f[e]);
            if (!(done >> e & 1) && have(e) && b > best) { best = b; at = index(e); slot = e; }    // indices rise with e
        }
        const unsigned m = lanes_max_u32<G>(best);
        const int who = (int)~lanes_max_u32<G>(best == m ? ~(unsigned)at : 0u);
        if (best == m && at == who) {
            done |= 1ull << slot;
            g.top_idx[row * g.k + j] = at;
            g.top_lp[row * g.k + j] = row_lp(r, order_value(m), g.inv_t);
        }
    }
}

// ---- gradient ---------------------------------------------------------------------------------------------------------------
// One walk, element-wise once the row's statistics are known: ln p = (x - m) / T - ln s, d = -p (g + h H + h ln p) / T, + g / T at the
// label.  A workgroup has 4 pieces per thread on their way before it computes: enough to keep memory busy, so rows are not persistent.
struct BwdRow {
    float m, log_s, q0, q1, dl;      // d = -p (q0 + q1 ln p), + dl at y
    int y;
    bool zero;                       // nothing but -inf, or nothing to differentiate: no label and no entropy, whatever the row holds
};
__device__ __forceinline__ BwdRow bwd_row(const ScoresBwd& g, long row) {
    BwdRow r;
    r.m = g.stat[2 * row];
    r.log_s = g.stat[2 * row + 1];
    r.y = g.labels ? g.labels[row] : -1;
    r.zero = (r.m == -INFINITY && r.log_s == 0.f) || (r.y < 0 && !g.d_ent);
    r.dl = g.d_lp && r.y >= 0 ? g.d_lp[row] * g.inv_t : 0.f;
    if (r.y >= g.V) r.dl = NAN;
    r.q1 = g.d_ent ? g.d_ent[row] * g.inv_t : 0.f;
    r.q0 = g.d_ent ? fmaf(r.q1, g.entropy[row], r.dl) : r.dl;
    return r;
}
template <class T> __device__ __forceinline__ void bwd_piece(const ScoresBwd& g, const BwdRow& r, const Raw16& d, T* o, int i0) {
    constexpr int E = Pack<T>::N;
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float lp = fmaf(elem<T>(d, e) - r.m, g.inv_t, -r.log_s), p = exp2_of(lp * LOG2E);
        f[e] = -p * fmaf(r.q1, fmaxf(lp, FAINT), r.q0);
    }
    if (r.y >= i0 && r.y < i0 + E)
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (i0 + e == r.y) f[e] += r.dl;
    if (r.zero)
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = 0.f;
    store_piece(o, i0, g.V, f, g.past);
}
// rows of many pieces: a workgroup takes U pieces per thread of one row
template <class T> __global__ __launch_bounds__(256) void scores_bwd_kernel(ScoresBwd g) {
    constexpr int E = Pack<T>::N, STEP = 256 * U * E;
    const long row = blockIdx.x / g.chunks;
    const int base = (int)(blockIdx.x - row * g.chunks) * STEP;
    const T* x = (const T*)g.X + row * g.ld;
    T* o = (T*)g.DX + row * g.lddx;
    Raw16 d[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int i0 = base + (j * 256 + (int)threadIdx.x) * E;
        if (i0 < g.V) d[j] = load_piece(x, i0, g.V, 0.f);
    }
    const BwdRow r = bwd_row(g, row);
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int i0 = base + (j * 256 + (int)threadIdx.x) * E;
        if (i0 < g.V) bwd_piece(g, r, d[j], o, i0);
    }
}
// short rows: one thread per piece, all rows' pieces in one run
template <class T> __global__ __launch_bounds__(256) void scores_bwd_few_kernel(ScoresBwd g) {
    constexpr int E = Pack<T>::N;
    const long p = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = p / g.chunks;
    if (row >= g.M) return;
    const int i0 = (int)(p - row * g.chunks) * E;
    const Raw16 d = load_piece((const T*)g.X + row * g.ld, i0, g.V, 0.f);
    bwd_piece(g, bwd_row(g, row), d, (T*)g.DX + row * g.lddx, i0);
}

constexpr int MAX_V = 1 << 23, MAX_K = 64;   // 64 parts of 32 fp32 steps

// Few classes stay in the registers of a team inside a wave: 16 lanes where they hold the row and a round per alternative is
// cheap (16384 x 100, top 64: 38.1 us in rounds of 16 lanes, 28 in the whole wave's list; top 5: 11.5 and 14.5).  Many
// rows up to 16384 (8192) classes take a wave each: no barriers, four times the rows in flight (16384 x 4000 bf16, top 5: 38.5 us
// instead of 65.7) -- unless most of 64 lanes would have only one group to find 64 alternatives in, for then the bound is too low
// and the list runs over (16384 x 2100, top 64: 346 us, 102 in a workgroup; top 48: 59 in a wave).  Beyond, a workgroup walks a row
// in steps of 4 pieces per thread (8192 16-bit or 4096 fp32 classes).  A row of more than 7 steps is split over workgroups (64 at most) where there are fewer than 512 rows: a join costs a launch (32000 bf16, top
// 20, us: 1 row 9.4 whole, 11.4 split; 600 rows 17.6, 22.0; 65000: 1 row 12.6, 11.4), and so is one whose group maxima would
// take more than 32 steps' room in LDS.
constexpr int FEW = 256;                  // lanes * pieces of the team form: up to 2048 16-bit or 1024 fp32 classes
constexpr int MOST_STEPS = 32, ALONE = 7;
constexpr int NARROW = 8, MANY = 2048;    // a wave per row: up to 8 of its steps, where there are rows enough for all CUs
struct ScoresShape {
    int splits, chunk, steps;             // splits = 0: the team form; -1: a wave per row
};
ScoresShape scores_shape(int M, int V, int dtype, int k) {
    const int E = elems_of(dtype);
    if (V <= FEW * E) return {0, V, 0};
    if (V <= NARROW * 64 * U * E && M >= MANY && (k <= 48 || V >= 72 * U * E)) return {-1, V, cdiv(V, 64 * U * E)};
    const int step = 256 * U * E, steps = cdiv(V, step);
    int S = M >= 512 || steps <= ALONE ? 1 : cdiv(1024, M > 0 ? M : 1);
    if (S > steps) S = steps;
    if (S > 64) S = 64;
    if (k > 0 && S * MOST_STEPS < steps) S = cdiv(steps, MOST_STEPS);
    const int each = cdiv(steps, S);
    return {cdiv(steps, each), each * step, each};
}

template <class T> int scores(Scores g, hipStream_t st) {
    constexpr int E = Pack<T>::N;
    const int dtype = sizeof(T) == 4 ? WFD_F32 : WFD_BF16;
    const ScoresShape s = scores_shape(g.M, g.V, dtype, g.k);
    g.splits = s.splits;
    g.chunk = s.chunk;
    if (s.splits == 0) {
#define WFD_FEW(G, R)                                                                                                    \
    if (g.V <= G * R * E && (G == 64 || g.k <= 16)) {                                                                    \
        if (!launchable(cdiv(g.M, 256 / G), 256)) return WFD_ERR_ARG;                                                    \
        hipLaunchKernelGGL((scores_few_kernel<T, G, R>), dim3(cdiv(g.M, 256 / G)), dim3(256), 0, st, g);                 \
        WFD_CHECK_LAUNCH();                                                                                              \
        return WFD_OK;                                                                                                   \
    }
        WFD_FEW(16, 1) WFD_FEW(16, 2) WFD_FEW(64, 1) WFD_FEW(64, 2) WFD_FEW(64, 4)
#undef WFD_FEW
    }
    if (s.splits < 0) {
        g.splits = 1;
        if (!launchable(g.M, 64)) return WFD_ERR_ARG;
        if (g.k > 0)
            hipLaunchKernelGGL((scores_kernel<T, 64, true>), dim3(g.M), dim3(64), (size_t)s.steps * 256, st, g);
        else
            hipLaunchKernelGGL((scores_kernel<T, 64, false>), dim3(g.M), dim3(64), 0, st, g);
        WFD_CHECK_LAUNCH();
        return WFD_OK;
    }
    const long parts = (long)g.M * s.splits;
    if (!launchable(parts, 256)) return WFD_ERR_ARG;
    if (g.k > 0)
        hipLaunchKernelGGL((scores_kernel<T, 256, true>), dim3((unsigned)parts), dim3(256), (size_t)s.steps * 1024, st, g);
    else
        hipLaunchKernelGGL((scores_kernel<T, 256, false>), dim3((unsigned)parts), dim3(256), 0, st, g);
    WFD_CHECK_LAUNCH();
    if (s.splits > 1) {
        hipLaunchKernelGGL((scores_join_kernel<T>), dim3(g.M), dim3(256), (size_t)s.splits * g.k * 8, st, g);
        WFD_CHECK_LAUNCH();
    }
    return WFD_OK;
}

template <class T> int scores_bwd(ScoresBwd g, hipStream_t st) {
    constexpr int E = Pack<T>::N, STEP = 256 * U * E;
    if (g.V > STEP / 2) {
        g.chunks = cdiv(g.V, STEP);
        const long blocks = (long)g.M * g.chunks;
        if (!launchable(blocks, 256)) return WFD_ERR_ARG;
        hipLaunchKernelGGL(scores_bwd_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, g);
    } else {
        g.chunks = cdiv(g.V, E);
        const long blocks = ((long)g.M * g.chunks + 255) / 256;
        if (!launchable(blocks, 256)) return WFD_ERR_ARG;
        hipLaunchKernelGGL(scores_bwd_few_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, g);
    }
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}

}  // namespace

extern "C" {

int wfd_label_scores_floats(int M, int V, int dtype, int k) {
    if (!wfd_dtype_ok(dtype) || M < 0 || V <= 0 || V > MAX_V || k < 0 || k > MAX_K || k > V) return -1;
    const ScoresShape s = scores_shape(M, V, dtype, k);
    if (M == 0 || s.splits <= 1) return 0;
    const long n = (long)M * s.splits * (3 + 2 * k);
    return n > 0x7fffffffL ? -1 : (int)n;
}

int wfd_label_scores(const void* logits, int ldl, int dtype, int M, int V, const int* labels, float temperature, int k,
                     float* logprob, float* entropy, float* stat, float* top_logprob, int* top_index, float* work,
                     void* stream) {
    const int need = wfd_label_scores_floats(M, V, dtype, k);
    if (need < 0 || (M > 0 && need > 0 && !work) || !(temperature >= 1e-6f) || !(temperature <= 1e6f)) return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if ((k > 0 && (!top_logprob || !top_index)) || (logprob && !labels)) return WFD_ERR_ARG;
    if (!rows_ok(logits, ldl, M, V, dtype)) return WFD_ERR_ARG;
    Scores g{logits, labels, logprob, entropy, stat, top_logprob, top_index, work, ldl, M, V, k, 1.f / temperature,
             log2e_over(temperature), 0, 0};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) return scores<float>(g, st);
    return dtype == WFD_BF16 ? scores<bf16_t>(g, st) : scores<f16_t>(g, st);
}

int wfd_label_scores_bwd(const void* logits, int ldl, int dtype, int M, int V, const int* labels, float temperature,
                         const float* stat, const float* entropy, const float* d_logprob, const float* d_entropy,
                         void* dlogits, int lddl, void* stream) {
    if (!wfd_dtype_ok(dtype) || M < 0 || V <= 0 || V > MAX_V || !(temperature >= 1e-6f) || !(temperature <= 1e6f))
        return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if ((d_logprob && !labels) || (d_entropy && !entropy)) return WFD_ERR_ARG;
    if (!stat || !rows_ok(logits, ldl, M, V, dtype) || !rows_ok(dlogits, lddl, M, V, dtype)) return WFD_ERR_ARG;
    if (!same_rows(dlogits, lddl, logits, ldl, M)) return WFD_ERR_ARG;
    ScoresBwd g{logits, labels, stat, entropy, d_logprob, d_entropy, dlogits, ldl, lddl, M, V, 1.f / temperature, 0,
                past_caches(M, V, dtype == WFD_F32 ? 4 : 2)};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) return scores_bwd<float>(g, st);
    return dtype == WFD_BF16 ? scores_bwd<bf16_t>(g, st) : scores_bwd<f16_t>(g, st);
}

}  // extern "C"
