// Token scores: for each row of logits x the log probability of a given token,
// the entropy and the most likely tokens.
//
//   m = max x,  S = sum e^(x - m),  W = sum (x - m) e^(x - m)
//   logprob(t) = x_t - m - log S,   H = log S - W / S
//
// Bound by HBM: every logit is read once.
#include "common.cuh"
#include "kernels.h"

namespace mlxd {

constexpr int SC_THREADS = 512, SC_TOP = 32;

struct ScoreCall {
    const void *x;
    int64_t stride;
    int rows, V, top;
    const int32_t *targets;
    float *lp, *ent, *tlp;
    int32_t *ids;
};

// order of the top list: larger logits first, NaN last, equal values (+0 and
// -0 too) by index
MLXD_DEV uint32_t sc_key(float v) {
    if (isnan(v)) return 0u;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
MLXD_DEV float sc_val(uint32_t k) {
    return k == 0u ? __int_as_float(0x7fc00000) : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename T>
MLXD_DEV float sc_load(const T *p, int i);
template <>
MLXD_DEV float sc_load<uint16_t>(const uint16_t *p, int i) { return bf2f(p[i]); }
template <>
MLXD_DEV float sc_load<float>(const float *p, int i) { return p[i]; }

template <typename T>
__global__ void __launch_bounds__(SC_THREADS) scores_kernel(ScoreCall c) {
    __shared__ unsigned long long s_key[SC_THREADS / 32];
    __shared__ double s_sum[SC_THREADS / 32][2];
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const T *x = (const T *)c.x + (int64_t)r * c.stride;
    auto best = [&](unsigned long long below) {
        unsigned long long b = 0;
        for (int i = tid; i < c.V; i += SC_THREADS) {
            const unsigned long long k = ((unsigned long long)sc_key(sc_load(x, i)) << 32) | (uint32_t)~i;
            if (k < below && k > b) b = k;
        }
        for (int o = 16; o; o >>= 1) b = max(b, __shfl_xor_sync(~0u, b, o));
        __syncthreads();
        if (lane == 0) s_key[warp] = b;
        __syncthreads();
        for (int w = 0; w < SC_THREADS / 32; w++) b = max(b, s_key[w]);
        return b;
    };
    const unsigned long long first = best(~0ull);
    const float m = sc_val((uint32_t)(first >> 32));
    const bool empty = m == -INFINITY;
    // S without the maximum's own term (1), so that log1p keeps small sums
    const int at = (int)~(uint32_t)first;
    double S = 0, W = 0;
    for (int i = tid; i < c.V; i += SC_THREADS) {
        if (i == at) continue;
        const float v = sc_load(x, i), e = empty ? 0.f : expf(v - m);
        S += e;
        if (e != 0.f) W += (double)e * (v - m);
    }
    for (int o = 16; o; o >>= 1) {
        S += __shfl_xor_sync(~0u, S, o);
        W += __shfl_xor_sync(~0u, W, o);
    }
    if (lane == 0) {
        s_sum[warp][0] = S;
        s_sum[warp][1] = W;
    }
    __syncthreads();
    S = W = 0;
    for (int w = 0; w < SC_THREADS / 32; w++) {
        S += s_sum[w][0];
        W += s_sum[w][1];
    }
    if (!(m < INFINITY)) S = nan("");   // +inf, or nothing but NaN
    const double ls = log1p(S);
    if (tid == 0) {
        const int t = c.targets ? c.targets[r] : 0;
        if (c.lp)
            c.lp[r] = t < 0 || t >= c.V ? __int_as_float(0x7fc00000)
                      : empty           ? -INFINITY
                                        : (float)((double)(sc_load(x, t) - m) - ls);
        if (c.ent) c.ent[r] = empty ? 0.f : (float)(ls - W / (1.0 + S));
    }
    unsigned long long k = first;
    for (int j = 0; j < c.top; j++) {
        if (j) k = best(k);
        if (tid == 0) {
            const float v = sc_val((uint32_t)(k >> 32));
            if (c.ids) c.ids[(int64_t)r * c.top + j] = (int32_t)~(uint32_t)k;
            if (c.tlp) c.tlp[(int64_t)r * c.top + j] = empty ? -INFINITY : (float)((double)(v - m) - ls);
        }
    }
}

}  // namespace mlxd

using namespace mlxd;

extern "C" int mlxd_cuda_token_scores(const void *logits, int dtype, int rows, int V, int64_t row_stride,
                                      const int32_t *targets, int n_top, float *logprobs, float *entropy,
                                      int32_t *top_ids, float *top_logprobs, void *stream) {
    if ((dtype != MLXD_BF16 && dtype != MLXD_F32) || rows < 0 || V <= 0 || row_stride < 0 || n_top < 0 ||
        n_top > SC_TOP || n_top > V) {
        set_error("token_scores: bad arguments (n_top: at most 32 and V)");
        return -1;
    }
    if (logprobs && !targets) {
        set_error("token_scores: logprobs without targets");
        return -1;
    }
    if (rows == 0) return 0;
    if (!on_device(logits, "token_scores: logits") || (targets && !on_device(targets, "token_scores: targets")) ||
        (logprobs && !on_device(logprobs, "token_scores: logprobs")) ||
        (entropy && !on_device(entropy, "token_scores: entropy")) ||
        (n_top && top_ids && !on_device(top_ids, "token_scores: top ids")) ||
        (n_top && top_logprobs && !on_device(top_logprobs, "token_scores: top logprobs")))
        return -1;
    ScoreCall c = {logits, row_stride, rows, V, n_top, targets, logprobs, entropy, top_logprobs, top_ids};
    if (dtype == MLXD_BF16) scores_kernel<uint16_t><<<rows, SC_THREADS, 0, (cudaStream_t)stream>>>(c);
    else scores_kernel<float><<<rows, SC_THREADS, 0, (cudaStream_t)stream>>>(c);
    MLXD_CHECK(cudaGetLastError());
    return 0;
}
