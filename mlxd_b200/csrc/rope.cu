// Rotary positions as a single op: y = x with the leading `dims` features of
// every head turned by their token's position.
//
//   u = a cos(p w) - b sin(p w),  v = a sin(p w) + b cos(p w)
//
// over the pairs (a, b) = (x_i, x_{i + dims/2}) or (x_2i, x_2i+1). The angle in
// turns, p * w / 2 pi, is reduced to [-1/2, 1/2] in f64 (f32 would lose the
// low bits of far positions: at p = 2^17 the fast pairs would be off by 2^-7
// turns), its sine and cosine are f32, the rotation is f32 and rounded once.
//
// Bound by HBM: x in, y out. A CTA first makes the cosines and sines of its
// tokens in shared memory, once per (token, pair) for all heads, then streams
// the heads.
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace mlxd {

constexpr int RP_THREADS = 256, RP_MAXPAIRS = 128, RP_MAXTOK = 4;

struct RopeCall {
    const void *x;
    void *y;
    int64_t xt, xh, yt, yh;    // token and head strides in elements
    const int32_t *pos;        // or null: pos0 + t
    int pos0, n, heads, dims, D;
    int tokens, hblock;        // tokens and heads per CTA
    float mag;
    double turns[RP_MAXPAIRS]; // turns per position
};

template <typename T>
MLXD_DEV float rp_get(T v);
template <>
MLXD_DEV float rp_get<uint16_t>(uint16_t v) { return bf2f(v); }
template <>
MLXD_DEV float rp_get<float>(float v) { return v; }
template <typename T>
MLXD_DEV T rp_put(float v);
template <>
MLXD_DEV uint16_t rp_put<uint16_t>(float v) { return f2bf(v); }
template <>
MLXD_DEV float rp_put<float>(float v) { return v; }

template <typename T, bool INTER>
__global__ void __launch_bounds__(RP_THREADS) rope_kernel(const __grid_constant__ RopeCall c) {
    __shared__ float2 cs[RP_MAXTOK][RP_MAXPAIRS];
    const int pairs = c.dims / 2;
    const int t0 = blockIdx.x * c.tokens, nt = min(c.tokens, c.n - t0);
    for (int i = threadIdx.x; i < nt * pairs; i += RP_THREADS) {
        const int t = i / pairs, j = i % pairs;
        const int p = c.pos ? c.pos[t0 + t] : c.pos0 + t0 + t;
        const double a = (double)p * c.turns[j];
        float si, co;
        sincospif((float)(2.0 * (a - rint(a))), &si, &co);
        cs[t][j] = make_float2(co * c.mag, si * c.mag);
    }
    __syncthreads();
    const int h0 = blockIdx.y * c.hblock, nh = min(c.hblock, c.heads - h0);
    const int per = pairs + (c.D - c.dims);   // rotated pairs and copied features of a head
    for (int i = threadIdx.x; i < nt * nh * per; i += RP_THREADS) {
        const int j = i % per, th = i / per, t = th / nh, h = h0 + th % nh;
        const T *x = (const T *)c.x + (t0 + t) * c.xt + h * c.xh;
        T *y = (T *)c.y + (t0 + t) * c.yt + h * c.yh;
        if (j < pairs) {
            const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : j + pairs;
            const float a = rp_get<T>(x[ia]), b = rp_get<T>(x[ib]);
            const float2 r = cs[t][j];
            y[ia] = rp_put<T>(a * r.x - b * r.y);
            y[ib] = rp_put<T>(a * r.y + b * r.x);
        } else {
            y[c.dims + j - pairs] = x[c.dims + j - pairs];
        }
    }
}

// turns per position of every pair and the magnitude; the llama3 rule is the
// model path's (llama3_freqs), YaRN blends per pair by how often it turns over
// the original context
static int rope_turns(const mlxd_rope &r, RopeCall &c) {
    const double theta = r.theta, d = r.dims, f = r.factor, lo = r.lo, hi = r.hi, om = r.orig_max;
    const bool scaled = r.scaling != MLXD_ROPE_DEFAULT;
    const bool banded = r.scaling == MLXD_ROPE_LLAMA3 || r.scaling == MLXD_ROPE_YARN;
    if (r.scaling < MLXD_ROPE_DEFAULT || r.scaling > MLXD_ROPE_YARN || !(theta > 1.0) || !isfinite(theta) ||
        (scaled && (!(f >= 1.0) || !isfinite(f))) || (banded && (!(lo > 0.0) || !(hi > lo) || !isfinite(hi) || om < 1)) ||
        (r.scaling == MLXD_ROPE_YARN && (!(r.magnitude >= 0.f) || !isfinite(r.magnitude)))) {
        set_error("rope: invalid base or scaling parameters");
        return -1;
    }
    double y0 = 0, y1 = 0;
    c.mag = 1.0f;
    if (r.scaling == MLXD_ROPE_YARN) {
        const double k = d / (2.0 * log(theta));
        y0 = fmax(floor(k * log(om / (hi * 2.0 * M_PI))), 0.0);
        y1 = fmin(ceil(k * log(om / (lo * 2.0 * M_PI))), d - 1.0);
        if (!(y1 - y0 >= 0.001)) y1 = y0 + 0.001;
        c.mag = r.magnitude > 0.f ? r.magnitude : (float)(0.1 * log(f) + 1.0);
    }
    for (int i = 0; i < r.dims / 2; i++) {
        double w = pow(theta, -2.0 * i / d);
        if (r.scaling == MLXD_ROPE_LINEAR) {
            w /= f;
        } else if (r.scaling == MLXD_ROPE_LLAMA3) {
            const double keep = fmin(fmax((om * w / (2.0 * M_PI) - lo) / (hi - lo), 0.0), 1.0);
            w *= (1.0 - keep) / f + keep;
        } else if (r.scaling == MLXD_ROPE_YARN) {
            const double far = fmin(fmax((i - y0) / (y1 - y0), 0.0), 1.0);
            w *= far / f + 1.0 - far;
        }
        c.turns[i] = w / (2.0 * M_PI);
    }
    return 0;
}

template <typename T>
static int rope_launch(const RopeCall &c, bool inter, cudaStream_t st) {
    dim3 grid((c.n + c.tokens - 1) / c.tokens, (c.heads + c.hblock - 1) / c.hblock);
    if (inter) rope_kernel<T, true><<<grid, RP_THREADS, 0, st>>>(c);
    else rope_kernel<T, false><<<grid, RP_THREADS, 0, st>>>(c);
    MLXD_CHECK(cudaGetLastError());
    return 0;
}

}  // namespace mlxd

using namespace mlxd;

extern "C" int mlxd_cuda_rope(const void *x, int dtype, int n, int heads, int head_dim, int64_t x_token_stride,
                              int64_t x_head_stride, const mlxd_rope *r, const int32_t *pos_dev, int pos, void *y,
                              int64_t y_token_stride, int64_t y_head_stride, void *stream) {
    if (!r || (dtype != MLXD_BF16 && dtype != MLXD_F32) || n < 0 || heads <= 0 || heads > 65535 || head_dim < 2 ||
        head_dim > 2 * RP_MAXPAIRS || r->dims < 0 || r->dims > head_dim || (r->dims & 1)) {
        set_error("rope: bad arguments (dims: even, at most head_dim <= 256)");
        return -1;
    }
    if (x_token_stride < 0 || x_head_stride < 0 || y_token_stride < 0 || y_head_stride < head_dim ||
        (n > 1 && y_token_stride < head_dim)) {
        set_error("rope: rows of y overlap");
        return -1;
    }
    if (!pos_dev && (int64_t)pos + n > INT32_MAX) {
        set_error("rope: position %d + %d tokens overflows", pos, n);
        return -1;
    }
    if (n == 0) return 0;
    RopeCall c;
    c.dims = r->dims;
    if (rope_turns(*r, c) || !on_device(x, "rope: x") || !on_device(y, "rope: y") ||
        (pos_dev && !on_device(pos_dev, "rope: positions")))
        return -1;
    c.x = x;
    c.y = y;
    c.xt = x_token_stride;
    c.xh = x_head_stride;
    c.yt = y_token_stride;
    c.yh = y_head_stride;
    c.pos = pos_dev;
    c.pos0 = pos;
    c.n = n;
    c.heads = heads;
    c.D = head_dim;
    c.tokens = 1;
    c.hblock = heads;
    const bool inter = r->interleaved != 0;
    return dtype == MLXD_BF16 ? rope_launch<uint16_t>(c, inter, (cudaStream_t)stream)
                              : rope_launch<float>(c, inter, (cudaStream_t)stream);
}
