// Scores of given labels over V classes: log probability, entropy and the k best alternatives of each row of logits, and the
// gradient of log probability and entropy.  With temperature T, m = max x, z = (x - m) / T, s = sum exp z:
//   logprob(y) = z_y - ln s,   H = ln s - (sum z exp z) / s,   p = exp z / s
//   d x_i = (1 / T) (g ([i = y] - p_i) - h p_i (ln p_i + H))
// Sums are fp32 about the row's own maximum; (m, ln s) stay apart in `stat`, so that differences to the maximum are exact.
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
    int ld, M, V, k;
    float inv_t;
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
};

// order of alternatives: larger value first (NaN before every number, -0 as 0), then the lower index
__device__ __forceinline__ unsigned order_bits(float v) {
    if (v != v) return 0xffffffffu;
    const unsigned u = __float_as_uint(v + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float v, int i) {
    return ((unsigned long long)order_bits(v) << 32) | (unsigned)~i;
}

__device__ __forceinline__ unsigned long long block_max_key(unsigned long long v, unsigned long long* slot) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slot[0];
    for (int i = 1; i < 4; ++i) v = slot[i] > v ? slot[i] : v;
    return v;
}

template <class T> __global__ __launch_bounds__(256) void scores_kernel(Scores g) {
    __shared__ float slot[3][8];
    __shared__ unsigned long long kslot[4];
    const long row = blockIdx.x;
    const T* x = (const T*)g.X + row * g.ld;
    const int t = threadIdx.x, V = g.V;
    float m = -INFINITY;
    for (int i = t; i < V; i += 256) m = fmaxf(m, to_f32(x[i]));
    m = team_max<256>(m, slot[0]);
    float s = 0.f, u = 0.f;
    for (int i = t; i < V; i += 256) {
        const float z = (to_f32(x[i]) - m) * g.inv_t, e = __expf(z);
        s += e;
        if (e != 0.f) u = fmaf(z, e, u);
    }
    const float2 su = team_sum2<256>(s, u, slot[1]);
    // -inf - -inf is NaN: a row of nothing but -inf has to be told from one that also holds a NaN
    const bool none = m == -INFINITY;
    int bad = 0;
    if (none)
        for (int i = t; i < V; i += 256) bad |= isnan(to_f32(x[i]));
    bad = __syncthreads_or(bad);
    const bool empty = none && !bad;
    const float log_s = empty ? 0.f : logf(su.x);
    if (t == 0) {
        if (g.stat) { g.stat[2 * row] = m; g.stat[2 * row + 1] = log_s; }
        if (g.entropy) g.entropy[row] = empty ? 0.f : log_s - su.y / su.x;
        if (g.labels && g.logprob) {
            const int y = g.labels[row];
            float lp = 0.f;
            if (y >= V) lp = NAN;
            else if (y >= 0) lp = empty ? -INFINITY : (to_f32(x[y]) - m) * g.inv_t - log_s;
            g.logprob[row] = lp;
        }
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < g.k; ++j) {
        unsigned long long best = 0;
        for (int i = t; i < V; i += 256) {
            const unsigned long long key = order_key(to_f32(x[i]), i);
            if (key < last && key > best) best = key;
        }
        last = block_max_key(best, kslot);
        if (t == 0) {
            const int i = (int)~(unsigned)last;
            g.top_idx[row * g.k + j] = i;
            g.top_lp[row * g.k + j] = empty ? -INFINITY : (to_f32(x[i]) - m) * g.inv_t - log_s;
        }
    }
}

template <class T> __global__ __launch_bounds__(256) void scores_bwd_kernel(ScoresBwd g) {
    const long row = blockIdx.x;
    const T* x = (const T*)g.X + row * g.ld;
    T* o = (T*)g.DX + row * g.lddx;
    const float m = g.stat[2 * row], log_s = g.stat[2 * row + 1];
    const bool empty = m == -INFINITY && log_s == 0.f;
    const int y = g.labels ? g.labels[row] : -1;
    float dl = g.d_lp && y >= 0 ? g.d_lp[row] : 0.f;
    if (y >= g.V) dl = NAN;
    const float dh = g.d_ent ? g.d_ent[row] : 0.f, H = g.d_ent ? g.entropy[row] : 0.f;
    for (int i = threadIdx.x; i < g.V; i += 256) {
        const float lp = (to_f32(x[i]) - m) * g.inv_t - log_s, p = __expf(lp);
        float d = -dl * p - (p != 0.f ? dh * p * (lp + H) : 0.f);
        if (i == y) d += dl;
        o[i] = from_f32<T>(empty ? 0.f : d * g.inv_t);
    }
}

bool rows_ok(const void* p, int ld, int M, int V, int dtype) {
    const uintptr_t align = dtype == WFD_F32 ? 3 : 1;
    return p && !((uintptr_t)p & align) && (M <= 1 || ld >= V);
}
constexpr int MAX_V = 1 << 28, MAX_K = 64;

}  // namespace

extern "C" {

int wfd_label_scores_floats(int M, int V, int dtype, int k) {
    if (!wfd_dtype_ok(dtype) || M < 0 || V <= 0 || V > MAX_V || k < 0 || k > MAX_K || k > V) return -1;
    return 0;
}

int wfd_label_scores(const void* logits, int ldl, int dtype, int M, int V, const int* labels, float temperature, int k,
                     float* logprob, float* entropy, float* stat, float* top_logprob, int* top_index, float* work,
                     void* stream) {
    const int need = wfd_label_scores_floats(M, V, dtype, k);
    if (need < 0 || (M > 0 && need > 0 && !work) || !(temperature > 0.f) || !(temperature < INFINITY)) return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if ((k > 0 && (!top_logprob || !top_index)) || (logprob && !labels)) return WFD_ERR_ARG;
    if (!rows_ok(logits, ldl, M, V, dtype)) return WFD_ERR_ARG;
    Scores g{logits, labels, logprob, entropy, stat, top_logprob, top_index, ldl, M, V, k, 1.f / temperature};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) hipLaunchKernelGGL(scores_kernel<float>, dim3(M), dim3(256), 0, st, g);
    else if (dtype == WFD_BF16) hipLaunchKernelGGL(scores_kernel<bf16_t>, dim3(M), dim3(256), 0, st, g);
    else hipLaunchKernelGGL(scores_kernel<f16_t>, dim3(M), dim3(256), 0, st, g);
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}

int wfd_label_scores_bwd(const void* logits, int ldl, int dtype, int M, int V, const int* labels, float temperature,
                         const float* stat, const float* entropy, const float* d_logprob, const float* d_entropy,
                         void* dlogits, int lddl, void* stream) {
    if (!wfd_dtype_ok(dtype) || M < 0 || V <= 0 || V > MAX_V || !(temperature > 0.f) || !(temperature < INFINITY))
        return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if ((d_logprob && !labels) || (d_entropy && !entropy)) return WFD_ERR_ARG;
    if (!stat || !rows_ok(logits, ldl, M, V, dtype) || !rows_ok(dlogits, lddl, M, V, dtype)) return WFD_ERR_ARG;
    ScoresBwd g{logits, labels, stat, entropy, d_logprob, d_entropy, dlogits, ldl, lddl, M, V, 1.f / temperature};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) hipLaunchKernelGGL(scores_bwd_kernel<float>, dim3(M), dim3(256), 0, st, g);
    else if (dtype == WFD_BF16) hipLaunchKernelGGL(scores_bwd_kernel<bf16_t>, dim3(M), dim3(256), 0, st, g);
    else hipLaunchKernelGGL(scores_bwd_kernel<f16_t>, dim3(M), dim3(256), 0, st, g);
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}

}  // extern "C"
