// Loss of a student that learns from a teacher's K top logits (and, mixed in, from a label), with its gradient.
// Teacher: entries j with index i_j and value t_j, q = softmax(t / T) over the entries that are there (index >= 0).
// Student row x over V classes, p = softmax(x / T), p1 = softmax(x):
//   loss = w T^2 sum_j q_j (ln q_j - ln p(i_j)) - u ln p1(y)
//   d x_i = r (w T (p_i [any entry] - sum_{j: i_j = i} q_j) + u (p1_i - [i = y]))          r = grad_scale * row_scale[row]
// An index that occurs twice counts twice.  No entry (or none above -inf): the first term is 0; y < 0: the second is 0.
// A row that holds nothing but -inf has loss +inf and gradient 0; an index or label >= V makes its row NaN.
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
    int ld, lddx, ldt, M, V, K;
    float temp, w, u, scale;
};

template <class T> __global__ __launch_bounds__(256) void distill_kernel(Distill g) {
    __shared__ float slot[6][8];
    __shared__ float q[MAX_ENTRIES];
    __shared__ int at[MAX_ENTRIES];
    const long row = blockIdx.x;
    const T* x = (const T*)g.X + row * g.ld;
    const int t = threadIdx.x, V = g.V, K = g.w != 0.f ? g.K : 0;
    const float it = 1.f / g.temp;
    const int y = g.u != 0.f && g.labels ? g.labels[row] : -1;
    float bad = y >= V ? 1.f : 0.f;
    int e_idx = -1;
    float e_val = -INFINITY, e_x = 0.f;
    if (t < K) {
        e_idx = g.t_idx[row * g.ldt + t];
        if (e_idx >= V) { bad = 1.f; e_idx = -1; }
        if (e_idx >= 0) { e_val = g.t_val[row * g.ldt + t]; e_x = to_f32(x[e_idx]); }
        at[t] = e_idx;
    }
    const float xy = y >= 0 && y < V ? to_f32(x[y]) : 0.f;
    float m = -INFINITY;
    for (int i = t; i < V; i += 256) m = fmaxf(m, to_f32(x[i]));
    m = team_max<256>(m, slot[0]);
    float s = 0.f, s1 = 0.f;
    for (int i = t; i < V; i += 256) {
        const float d = to_f32(x[i]) - m;
        s += __expf(d * it);
        s1 += __expf(d);
    }
    const float2 ss = team_sum2<256>(s, s1, slot[1]);
    int nan_here = 0;
    if (m == -INFINITY)
        for (int i = t; i < V; i += 256) nan_here |= isnan(to_f32(x[i]));
    const bool empty = m == -INFINITY && !__syncthreads_or(nan_here);
    const float log_s = logf(ss.x), log_s1 = logf(ss.y);
    // the teacher's softmax
    const float tm = team_max<256>(e_val, slot[2]);
    const float e = e_val == -INFINITY ? 0.f : __expf((e_val - tm) * it);
    const float2 es = team_sum2<256>(e, bad, slot[3]);
    const bool taught = !(es.x <= 0.f);
    const float my_q = taught ? e / es.x : 0.f;
    if (t < K) q[t] = my_q;
    float term = 0.f;
    if (my_q != 0.f) {
        const float lp = empty ? -INFINITY : (e_x - m) * it - log_s;
        term = my_q * ((e_val - tm) * it - logf(es.x) - lp);
    }
    const float kl = team_sum<256>(term, slot[4]);
    const bool wrong = es.y != 0.f;
    if (t == 0) {
        float loss = g.w != 0.f ? g.w * g.temp * g.temp * kl : 0.f;
        if (y >= 0) loss -= g.u * (empty ? -INFINITY : xy - m - log_s1);
        g.loss[row] = wrong ? NAN : loss;
    }
    if (!g.DX) return;
    T* o = (T*)g.DX + row * g.lddx;
    float r = g.scale * (g.row_scale ? g.row_scale[row] : 1.f);
    if (wrong) r = NAN;
    const float cw = taught ? r * g.w * g.temp / ss.x : 0.f, cu = y >= 0 ? r * g.u / ss.y : 0.f;
    for (int i = t; i < V; i += 256) {
        const float d = to_f32(x[i]) - m;
        float v = 0.f;
        if (cw != 0.f) v = cw * __expf(d * it);
        if (cu != 0.f) v = fmaf(cu, __expf(d), v);
        if (i == y) v -= r * g.u;
        if (empty) v = wrong ? NAN : 0.f;
        bool entry = false;
        float sq = 0.f;
        for (int j = 0; j < K; ++j)
            if (at[j] == i) { entry = true; sq += q[j]; }
        if (entry && !empty) v -= r * g.w * g.temp * sq;
        o[i] = from_f32<T>(v);
    }
}

bool rows_ok(const void* p, int ld, int M, int V, int dtype) {
    const uintptr_t align = dtype == WFD_F32 ? 3 : 1;
    return p && !((uintptr_t)p & align) && (M <= 1 || ld >= V);
}
constexpr int MAX_V = 1 << 28;

}  // namespace

extern "C" {

int wfd_distill_floats(int M, int V, int dtype) {
    if (!wfd_dtype_ok(dtype) || M < 0 || V <= 0 || V > MAX_V) return -1;
    return 0;
}

int wfd_distill(const void* logits, int ldl, int dtype, int M, int V, const int* t_index, const float* t_value, int ldt, int K,
                const int* labels, float temperature, float weight, float label_weight, const float* row_scale,
                float grad_scale, float* loss, void* dlogits, int lddl, float* work, void* stream) {
    const int need = wfd_distill_floats(M, V, dtype);
    if (need < 0 || (M > 0 && need > 0 && !work) || K < 0 || K > MAX_ENTRIES || !(temperature > 0.f) || !(temperature < INFINITY))
        return WFD_ERR_ARG;
    if (!(weight - weight == 0.f) || !(label_weight - label_weight == 0.f)) return WFD_ERR_ARG;
    if (M == 0) return WFD_OK;
    if (label_weight != 0.f && !labels) return WFD_ERR_ARG;
    if (!loss || !rows_ok(logits, ldl, M, V, dtype) || (dlogits && !rows_ok(dlogits, lddl, M, V, dtype))) return WFD_ERR_ARG;
    if (K > 0 && (!t_index || !t_value || (M > 1 && ldt < K))) return WFD_ERR_ARG;
    Distill g{logits, t_index, t_value, labels, row_scale, loss, dlogits, ldl, lddl, ldt, M, V, K, temperature, weight,
              label_weight, grad_scale};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == WFD_F32) hipLaunchKernelGGL(distill_kernel<float>, dim3(M), dim3(256), 0, st, g);
    else if (dtype == WFD_BF16) hipLaunchKernelGGL(distill_kernel<bf16_t>, dim3(M), dim3(256), 0, st, g);
    else hipLaunchKernelGGL(distill_kernel<f16_t>, dim3(M), dim3(256), 0, st, g);
    WFD_CHECK_LAUNCH();
    return WFD_OK;
}

}  // extern "C"
