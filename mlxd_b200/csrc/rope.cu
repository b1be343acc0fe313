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
// the heads. 8192 tokens x 72 heads of 128 in bf16: 54 us, 85% of the measured
// copy rate; 8 CTAs of 256 threads to an SM hide the loads' latency (4: 67 us,
// 6: 60). Rows that do not come in whole vectors go an element at a time: the
// same prompt at an odd stride 165 us, 8192 x 32 heads of 80 with 40 turned 63 us
// (floor 12.8). A launch of one token is latency alone (2.6 us).
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
    int per;                   // items of a head
    unsigned per_mul, h_mul;   // ceil(2^32 / per), ceil(2^32 / hblock) (0: divisor 1)
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

// N elements of a row: one 16-byte access, or one element
template <typename T, int N>
struct alignas(N * sizeof(T)) RopeVec {
    T e[N];
};

// An item is N pairs of one head (or N copied features): N = 8 (bf16) or 4 (f32)
// when every row starts on 16 bytes and the pairs and the copied rest come in
// whole vectors, else 1. Items run over (token, head, vector) with the
// vector fastest, so that a warp's accesses are contiguous.
template <typename T, bool INTER, int N>
__global__ void __launch_bounds__(RP_THREADS, 8) rope_kernel(const __grid_constant__ RopeCall c) {
    __shared__ __align__(16) float2 cs[RP_MAXTOK][RP_MAXPAIRS];
    using V = RopeVec<T, N>;
    const int pairs = c.dims / 2, nrot = pairs / N;
    const int t0 = blockIdx.x * c.tokens, nt = min(c.tokens, c.n - t0);
    const int h0 = blockIdx.y * c.hblock, nh = min(c.hblock, c.heads - h0);
    const int items = nt * nh * c.per;
    struct At {
        const T *x;
        T *y;
        int j, t;
    };
    auto at = [&](int i) {
        const int th = __umulhi(i, c.per_mul) + (c.per_mul ? 0 : i), t = nt == 1 ? 0 : __umulhi(th, c.h_mul) + (c.h_mul ? 0 : th);
        const int h = h0 + th - t * nh;
        return At{(const T *)c.x + (t0 + t) * c.xt + h * c.xh, (T *)c.y + (t0 + t) * c.yt + h * c.yh, i - th * c.per, t};
    };
    // feature of the first and second vector of item j
    auto first = [&](int j) { return j < nrot ? (INTER ? 2 * N * j : N * j) : c.dims + N * (j - nrot); };
    const int second = INTER ? N : pairs;
    for (int i = threadIdx.x; i < nt * pairs; i += RP_THREADS) {
        const int t = nt == 1 ? 0 : i / pairs, j = i - t * pairs;
        const int p = c.pos ? c.pos[t0 + t] : c.pos0 + t0 + t;
        const double g = (double)p * c.turns[j];
        float si, co;
        sincospif((float)(2.0 * (g - rint(g))), &si, &co);
        // element e of vector v at e * nrot + v: a warp's reads meet no bank twice
        cs[t][j % N * nrot + j / N] = make_float2(co * c.mag, si * c.mag);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < items; i += RP_THREADS) {
        const At p = at(i);
        const int f = first(p.j);
        const V a = *reinterpret_cast<const V *>(p.x + f);
        if (p.j >= nrot) {
            *reinterpret_cast<V *>(p.y + f) = a;
            continue;
        }
        const V b = *reinterpret_cast<const V *>(p.x + f + second);
        T in[2 * N], out[2 * N];                     // pair e: in[ia(e)], in[ib(e)]
        auto ia = [](int e) { return INTER ? 2 * e : e; };
        auto ib = [](int e) { return INTER ? 2 * e + 1 : N + e; };
#pragma unroll
        for (int e = 0; e < N; e++) {
            in[e] = a.e[e];
            in[N + e] = b.e[e];
        }
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float2 r = cs[p.t][e * nrot + p.j];
            const float u = rp_get<T>(in[ia(e)]), v = rp_get<T>(in[ib(e)]);
            out[ia(e)] = rp_put<T>(u * r.x - v * r.y);
            out[ib(e)] = rp_put<T>(u * r.y + v * r.x);
        }
        V ra, rb;
#pragma unroll
        for (int e = 0; e < N; e++) {
            ra.e[e] = out[e];
            rb.e[e] = out[N + e];
        }
        *reinterpret_cast<V *>(p.y + f) = ra;
        *reinterpret_cast<V *>(p.y + f + second) = rb;
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

// i / d = umulhi(i, ceil(2^32 / d)) for i and d below 2^16 (the items of a CTA)
static unsigned divisor(int d) { return d == 1 ? 0u : (unsigned)((0x100000000ull + d - 1) / d); }

template <typename T, int N>
static int rope_launch(RopeCall &c, bool inter, cudaStream_t st) {
    c.per = c.dims / 2 / N + (c.D - c.dims) / N;
    // Few tokens: the heads of one over CTAs of up to two items a thread
    // (latency). CTAs enough for all SMs several times over: all heads of a
    // token in one, or of up to 4 tokens (its cosines are made once). A CTA has
    // below 2^16 items (the divisions), of several tokens only with all their heads.
    const int two = 2 * RP_THREADS;
    c.tokens = 1;
    c.hblock = c.heads;
    if (c.n < 4 * num_sms()) {
        const int hb = (c.heads * c.per + two - 1) / two;
        c.hblock = (c.heads + hb - 1) / hb;
    } else {
        while (c.tokens < RP_MAXTOK && c.n / (c.tokens * 2) >= 4 * num_sms() &&
               (int64_t)c.tokens * 2 * c.heads * c.per <= 65535)
            c.tokens *= 2;
    }
    if ((int64_t)c.hblock * c.per > 65535) c.hblock = 65535 / c.per;
    const int hb = (c.heads + c.hblock - 1) / c.hblock;
    c.per_mul = divisor(c.per);
    c.h_mul = divisor(c.hblock);
    dim3 grid((c.n + c.tokens - 1) / c.tokens, hb);
    if (inter) rope_kernel<T, true, N><<<grid, RP_THREADS, 0, st>>>(c);
    else rope_kernel<T, false, N><<<grid, RP_THREADS, 0, st>>>(c);
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
    // y's rows do not overlap: heads within a token's span, or tokens within a head's
    const int64_t D = head_dim, most = INT64_MAX / 4 / ((int64_t)n + heads);
    const bool in_range = x_token_stride >= 0 && x_head_stride >= 0 && y_token_stride >= 0 && y_head_stride >= 0 &&
                          x_token_stride <= most && x_head_stride <= most && y_token_stride <= most && y_head_stride <= most;
    if (!in_range || !(((heads == 1 || y_head_stride >= D) &&
                        (n <= 1 || y_token_stride - D >= (heads - 1) * y_head_stride)) ||
                       ((n <= 1 || y_token_stride >= D) &&
                        (heads == 1 || y_head_stride - D >= (n - 1) * y_token_stride)))) {
        set_error("rope: rows of y overlap, or a stride out of range");
        return -1;
    }
    if (!pos_dev && (int64_t)pos + n > INT32_MAX) {
        set_error("rope: position %d + %d tokens overflows", pos, n);
        return -1;
    }
    if (n == 0) return 0;
    const int elem = dtype == MLXD_BF16 ? 2 : 4;
    RopeCall c;
    c.dims = r->dims;
    if (rope_turns(*r, c) || !on_device(x, "rope: x", elem) || !on_device(y, "rope: y", elem) ||
        (pos_dev && !on_device(pos_dev, "rope: positions", 4)))
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
    const bool inter = r->interleaved != 0;
    const int vec = dtype == MLXD_BF16 ? 8 : 4;
    const bool whole = c.dims % (2 * vec) == 0 && (c.D - c.dims) % vec == 0 && ((uintptr_t)x & 15) == 0 &&
                       ((uintptr_t)y & 15) == 0 && (c.xt | c.xh | c.yt | c.yh) % vec == 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == MLXD_BF16) return whole ? rope_launch<uint16_t, 8>(c, inter, st) : rope_launch<uint16_t, 1>(c, inter, st);
    return whole ? rope_launch<float, 4>(c, inter, st) : rope_launch<float, 1>(c, inter, st);
}
