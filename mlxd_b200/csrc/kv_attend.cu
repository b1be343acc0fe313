// Attention over the rows of a cache layer, and of a batch that shares a
// prefix, for callers that drive layers themselves.
//
//   out_i = sum_j e^(s (q_i . k_j) - m_i) v_j / sum_j e^(s (q_i . k_j) - m_i)
//
// over the keys j <= p_i with p_i - j < window or j < sinks, in one pass over
// the keys with a running maximum m_i.
#include <math.h>
#include <new>

#include "common.cuh"
#include "kernels.h"

namespace mlxd {

struct AttnCall {
    const uint16_t *q;
    uint16_t *out;
    int64_t q_stride, out_stride;
    int n, hq, hkv, D, rep;
    int window, sinks;
    float scale;
    const uint16_t *k, *v;     // the layer's rows [hkv][cap][D]
    int cap, ring_sinks;       // slot of position p: p below cap, else in the ring above ring_sinks
    int pos0;                  // cache call: position of query 0
    // group call: one query per sequence
    const int32_t *lens;       // null: cache call
    const uint16_t *tk, *tv;   // tails [n][hkv][tcap][D]
    int tcap, prefix;
};

// One warp per (query, head): lane l holds features 8 l .. 8 l + 7; a dot
// product per key, reduced over the lanes. Serves every head_dim.
__global__ void __launch_bounds__(128) attend_rows_kernel(AttnCall c) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)c.n * c.hq) return;
    const int i = (int)(row / c.hq), h = (int)(row % c.hq), g = h / c.rep;
    int p = c.pos0 + i;
    if (c.lens) {
        const int len = min(c.lens[i], c.tcap);
        if (len < 0) return;
        p = c.prefix + len - 1;
    }
    const bool mine = lane * 8 < c.D;
    float q[8], acc[8], m = -INFINITY, l = 0.f;
    for (int d = 0; d < 8; d++) {
        q[d] = mine ? bf2f(c.q[i * c.q_stride + (int64_t)h * c.D + lane * 8 + d]) * c.scale : 0.f;
        acc[d] = 0.f;
    }
    const int lo = c.window ? max(0, p - c.window + 1) : 0;
    const int head = c.window ? min(c.sinks, lo) : 0;   // sinks before the window
    for (int t = 0; t < head + p + 1 - lo; t++) {
        const int j = t < head ? t : lo + t - head;
        const uint16_t *kr, *vr;
        if (c.lens && j >= c.prefix) {
            const int64_t o = (((int64_t)i * c.hkv + g) * c.tcap + (j - c.prefix)) * c.D;
            kr = c.tk + o;
            vr = c.tv + o;
        } else {
            const int s = j < c.cap ? j : c.ring_sinks + (j - c.ring_sinks) % (c.cap - c.ring_sinks);
            const int64_t o = ((int64_t)g * c.cap + s) * c.D;
            kr = c.k + o;
            vr = c.v + o;
        }
        float z = 0.f;
        if (mine)
            for (int d = 0; d < 8; d++) z = fmaf(q[d], bf2f(kr[lane * 8 + d]), z);
        z = warp_sum(z);
        const float mn = fmaxf(m, z), a = mn == -INFINITY ? 1.f : expf(m - mn), e = mn == -INFINITY ? 0.f : expf(z - mn);
        m = mn;
        l = fmaf(l, a, e);
        if (mine)
            for (int d = 0; d < 8; d++) acc[d] = fmaf(acc[d], a, e * bf2f(vr[lane * 8 + d]));
    }
    if (mine)
        for (int d = 0; d < 8; d++)
            c.out[i * c.out_stride + (int64_t)h * c.D + lane * 8 + d] = f2bf(l > 0.f ? acc[d] / l : l);
}

// tail rows of one decode step: sequence blockIdx.x
__global__ void group_append_kernel(const uint16_t *__restrict__ k, int64_t ks, const uint16_t *__restrict__ v,
                                    int64_t vs, const int32_t *__restrict__ lens, uint16_t *tk, uint16_t *tv, int hkv,
                                    int cap, int D) {
    const int i = blockIdx.x, len = lens[i];
    if (len < 1 || len > cap) return;
    for (int e = threadIdx.x; e < hkv * D / 8; e += blockDim.x) {
        const int h = e / (D / 8), d = e % (D / 8);
        const int64_t o = (((int64_t)i * hkv + h) * cap + len - 1) * D;
        reinterpret_cast<uint4 *>(tk + o)[d] = reinterpret_cast<const uint4 *>(k + i * ks)[e];
        reinterpret_cast<uint4 *>(tv + o)[d] = reinterpret_cast<const uint4 *>(v + i * vs)[e];
    }
}

static int attend(const AttnCall &c, void *ws, size_t ws_bytes, cudaStream_t st) {
    const int64_t rows = (int64_t)c.n * c.hq;
    if ((rows + 3) / 4 > INT32_MAX) {
        set_error("attention: too many query rows");
        return -1;
    }
    attend_rows_kernel<<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(c);
    MLXD_CHECK(cudaGetLastError());
    return 0;
}

// the checks that both calls share; fills the call's common half
static int attn_call(AttnCall &c, const char *what, int hkv, int D, const void *q, int64_t q_stride, int n,
                     const mlxd_attn *a, void *out, int64_t out_stride, const void *ws, size_t ws_bytes) {
    if (!a || a->n_heads <= 0 || a->n_heads % hkv || a->window < 0 || a->sinks < 0 || !(a->scale >= 0.f) ||
        !isfinite(a->scale)) {
        set_error("%s: bad attention parameters (heads a multiple of %d, window and sinks not negative, scale finite)",
                  what, hkv);
        return -1;
    }
    const int64_t row = (int64_t)a->n_heads * D;
    if (q_stride < row || out_stride < row || q_stride % 8 || out_stride % 8 || ((uintptr_t)q & 15) ||
        ((uintptr_t)out & 15)) {
        set_error("%s: rows of q and out need 16-byte alignment and strides of at least %lld elements", what,
                  (long long)row);
        return -1;
    }
    if (ws_bytes < mlxd_cuda_attn_workspace_bytes(D) || ((uintptr_t)ws & 255)) {
        set_error("%s: workspace too small or misaligned", what);
        return -1;
    }
    if (!on_device(q, "attention: q") || !on_device(out, "attention: out") || !on_device(ws, "attention: workspace"))
        return -1;
    c.q = (const uint16_t *)q;
    c.out = (uint16_t *)out;
    c.q_stride = q_stride;
    c.out_stride = out_stride;
    c.n = n;
    c.hq = a->n_heads;
    c.hkv = hkv;
    c.D = D;
    c.rep = a->n_heads / hkv;
    c.window = a->window;
    c.sinks = a->window ? a->sinks : 0;
    c.scale = a->scale > 0.f ? a->scale : (float)(1.0 / sqrt((double)D));
    return 0;
}

static bool same_device(int device, const char *what) {
    int dev = 0;
    if (!cuda_ok(cudaGetDevice(&dev), what)) return false;
    if (dev != device) {
        set_error("%s: cache of device %d, the current device is %d", what, device, dev);
        return false;
    }
    return true;
}

}  // namespace mlxd

using namespace mlxd;

extern "C" {

size_t mlxd_cuda_attn_workspace_bytes(int head_dim) {
    if (head_dim <= 0) return 0;
    return 256;
}

int mlxd_cuda_kv_attend(const mlxd_kv *kv, int layer, const void *q, int64_t q_stride, int n, int pos,
                        const mlxd_attn *a, void *out, int64_t out_stride, void *ws, size_t ws_bytes, void *stream) {
    if (!kv || layer < 0 || layer >= kv->layers || n < 0 || pos < 0 || (int64_t)pos + n > INT32_MAX) {
        set_error("kv_attend: bad arguments");
        return -1;
    }
    if (kv->d % 8 || kv->d > 256) {
        set_error("kv_attend: head dim %d is not a multiple of 8 up to 256", kv->d);
        return -1;
    }
    if (n == 0) return 0;
    AttnCall c = {};
    if (attn_call(c, "kv_attend", kv->hkv, kv->d, q, q_stride, n, a, out, out_stride, ws, ws_bytes)) return -1;
    const int total = pos + n;
    if (total > kv->cap) {
        const int ring = kv->cap - kv->sinks;
        if (kv->window <= 0 || c.window <= 0 || (int64_t)n + c.window - 1 > ring) {
            set_error("kv_attend: positions up to %d with window %d are not held by a cache of %d rows (ring of %d)",
                      total, c.window, kv->cap, kv->window > 0 ? ring : 0);
            return -1;
        }
        if (c.sinks > kv->sinks) {
            set_error("kv_attend: %d sinks, the cache keeps %d", c.sinks, kv->sinks);
            return -1;
        }
    }
    if (!same_device(kv->device, "kv_attend")) return -1;
    const size_t layer_elems = (size_t)kv->hkv * kv->cap * kv->d;
    c.k = kv->k + layer * layer_elems;
    c.v = kv->v + layer * layer_elems;
    c.cap = kv->cap;
    c.ring_sinks = kv->sinks;
    c.pos0 = pos;
    return attend(c, ws, ws_bytes, (cudaStream_t)stream);
}

int mlxd_cuda_kv_group_create(mlxd_kv_group **out, const mlxd_kv *prefix, int prefix_len, int n_seqs,
                              int tail_capacity) {
    if (!out || !prefix || prefix_len < 0 || prefix_len > prefix->cap || n_seqs <= 0 || tail_capacity <= 0 ||
        (int64_t)prefix_len + tail_capacity > INT32_MAX || prefix->d % 8 || prefix->d > 256) {
        set_error("kv_group_create: bad arguments");
        return -1;
    }
    if (!same_device(prefix->device, "kv_group_create")) return -1;
    mlxd_kv_group *g = new (std::nothrow) mlxd_kv_group();
    if (!g) {
        set_error("kv_group_create: out of host memory");
        return -1;
    }
    g->prefix = prefix;
    g->prefix_len = prefix_len;
    g->n = n_seqs;
    g->cap = tail_capacity;
    g->layers = prefix->layers;
    g->hkv = prefix->hkv;
    g->d = prefix->d;
    g->device = prefix->device;
    const size_t bytes = (size_t)g->layers * n_seqs * g->hkv * tail_capacity * g->d * 2;
    if (!(g->k = (uint16_t *)dev_alloc(bytes)) || !(g->v = (uint16_t *)dev_alloc(bytes))) {
        mlxd_cuda_kv_group_destroy(g);
        return -1;
    }
    *out = g;
    return 0;
}

void mlxd_cuda_kv_group_destroy(mlxd_kv_group *g) {
    if (!g) return;
    cudaDeviceSynchronize();
    dev_free(g->k);
    dev_free(g->v);
    delete g;
}

int mlxd_cuda_kv_group_write(mlxd_kv_group *g, int layer, int seq, int row, int n, const void *k_dev,
                             const void *v_dev, void *stream) {
    if (!g || layer < 0 || layer >= g->layers || seq < 0 || seq >= g->n || row < 0 || n < 0 || n > g->cap - row) {
        set_error("kv_group_write: bad arguments");
        return -1;
    }
    if (n == 0) return 0;
    if (!on_device(k_dev, "kv_group_write: k") || !on_device(v_dev, "kv_group_write: v") ||
        !same_device(g->device, "kv_group_write"))
        return -1;
    const size_t rb = (size_t)g->d * 2;
    const size_t o = ((((size_t)layer * g->n + seq) * g->hkv) * g->cap + row) * g->d;
    MLXD_CHECK(cudaMemcpy2DAsync(g->k + o, g->cap * rb, k_dev, n * rb, n * rb, g->hkv, cudaMemcpyDeviceToDevice,
                                 (cudaStream_t)stream));
    MLXD_CHECK(cudaMemcpy2DAsync(g->v + o, g->cap * rb, v_dev, n * rb, n * rb, g->hkv, cudaMemcpyDeviceToDevice,
                                 (cudaStream_t)stream));
    return 0;
}

int mlxd_cuda_kv_group_append(mlxd_kv_group *g, int layer, const void *k, int64_t k_stride, const void *v,
                              int64_t v_stride, const int32_t *lens_dev, void *stream) {
    if (!g || layer < 0 || layer >= g->layers) {
        set_error("kv_group_append: bad arguments");
        return -1;
    }
    const int64_t row = (int64_t)g->hkv * g->d;
    if (k_stride < row || v_stride < row || k_stride % 8 || v_stride % 8 || ((uintptr_t)k & 15) || ((uintptr_t)v & 15)) {
        set_error("kv_group_append: rows need 16-byte alignment and strides of at least %lld elements", (long long)row);
        return -1;
    }
    if (!on_device(k, "kv_group_append: k") || !on_device(v, "kv_group_append: v") ||
        !on_device(lens_dev, "kv_group_append: lengths") || !same_device(g->device, "kv_group_append"))
        return -1;
    const size_t o = (size_t)layer * g->n * g->hkv * g->cap * g->d;
    group_append_kernel<<<g->n, 128, 0, (cudaStream_t)stream>>>((const uint16_t *)k, k_stride, (const uint16_t *)v,
                                                                v_stride, lens_dev, g->k + o, g->v + o, g->hkv, g->cap,
                                                                g->d);
    MLXD_CHECK(cudaGetLastError());
    return 0;
}

int mlxd_cuda_kv_group_attend(const mlxd_kv_group *g, int layer, const void *q, int64_t q_stride,
                              const int32_t *lens_dev, const mlxd_attn *a, void *out, int64_t out_stride, void *ws,
                              size_t ws_bytes, void *stream) {
    if (!g || layer < 0 || layer >= g->layers) {
        set_error("kv_group_attend: bad arguments");
        return -1;
    }
    AttnCall c = {};
    if (attn_call(c, "kv_group_attend", g->hkv, g->d, q, q_stride, g->n, a, out, out_stride, ws, ws_bytes) ||
        !on_device(lens_dev, "kv_group_attend: lengths") || !same_device(g->device, "kv_group_attend"))
        return -1;
    const size_t layer_elems = (size_t)g->hkv * g->prefix->cap * g->d;
    const size_t o = (size_t)layer * g->n * g->hkv * g->cap * g->d;
    c.k = g->prefix->k + layer * layer_elems;
    c.v = g->prefix->v + layer * layer_elems;
    c.cap = g->prefix->cap;
    c.lens = lens_dev;
    c.tk = g->k + o;
    c.tv = g->v + o;
    c.tcap = g->cap;
    c.prefix = g->prefix_len;
    return attend(c, ws, ws_bytes, (cudaStream_t)stream);
}

}  // extern "C"
