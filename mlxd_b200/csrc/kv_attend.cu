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

constexpr float LOG2E = 1.4426950408889634f;

struct AttnCall {
    const uint16_t *q;
    uint16_t *out;
    int64_t q_stride, out_stride;
    int n, hq, hkv, D, rep;
    int window, sinks;         // window 0: none
    float scale;
    const uint16_t *k, *v;     // the layer's rows [hkv][cap][D]
    int cap, ring_sinks;       // slot of position p: p below cap, else in the ring above ring_sinks
    int total;                 // positions written
    int pos0;                  // cache call: position of query 0
    // group call: one query per sequence
    const int32_t *lens;       // null: cache call
    const uint16_t *tk, *tv;   // tails [n][hkv][tcap][D]
    int tcap, prefix;
    // results of the prefix half: per (split, query row) m and l, o [D]
    const float *part_o;
    const float2 *part_ml;
    int parts;
};

// position of query token i (group: -1 when nothing of it is asked)
MLXD_DEV int query_pos(const AttnCall &c, int i) {
    if (!c.lens) return c.pos0 + i;
    const int len = min(c.lens[i], c.tcap);
    return len < 0 ? -1 : c.prefix + len - 1;
}
MLXD_DEV int window_lo(const AttnCall &c, int p) { return c.window ? max(0, p - c.window + 1) : 0; }

// The slots that hold positions [lo, hi) and the sinks below lo: [0, a1),
// [c0, c1) (the wrapped end of a ring) and [b0, b1), ascending. In a wrapped
// ring [lo, hi) lies above the kept sinks and spans at most the ring.
struct Span {
    int a1, c0, c1, b0, b1;
};
MLXD_DEV Span span_of(const AttnCall &c, int lo, int hi) {
    Span s;
    s.a1 = min(c.sinks, lo);
    if (c.total <= c.cap) {
        s.b0 = lo;
        s.b1 = min(hi, c.total);
        s.c0 = s.c1 = 0;
    } else {
        const int ring = c.cap - c.ring_sinks, x = (lo - c.ring_sinks) % ring, len = hi - lo;
        s.b0 = c.ring_sinks + x;
        s.b1 = min(s.b0 + len, c.cap);
        s.c0 = c.ring_sinks;
        s.c1 = c.ring_sinks + max(0, x + len - ring);
    }
    return s;
}
// position in slot s of a cache that holds positions [0, total)
MLXD_DEV int slot_pos(const AttnCall &c, int s) {
    if (c.total <= c.cap || s < c.ring_sinks) return s;
    const int ring = c.cap - c.ring_sinks, last = c.total - 1, d = (last - c.ring_sinks) % ring - (s - c.ring_sinks);
    return last - (d >= 0 ? d : d + ring);
}

// One warp per (query, head): lane l holds features 8 l .. 8 l + 7; a dot
// product per key, reduced over the lanes. Serves every head_dim.
__global__ void __launch_bounds__(128) attend_rows_kernel(AttnCall c) {
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)c.n * c.hq) return;
    const int i = (int)(row / c.hq), h = (int)(row % c.hq), g = h / c.rep;
    if (c.lens && c.lens[i] < 0) return;
    const int p = query_pos(c, i);
    const bool mine = lane * 8 < c.D;
    float q[8], acc[8], m = -INFINITY, l = 0.f;
    for (int d = 0; d < 8; d++) {
        q[d] = mine ? bf2f(c.q[i * c.q_stride + (int64_t)h * c.D + lane * 8 + d]) * c.scale : 0.f;
        acc[d] = 0.f;
    }
    const int lo = window_lo(c, p), head = min(c.sinks, lo);   // sinks before the window
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

// ---- few query rows per kv head (single tokens, tails): key-split warps
//
// Up to 16 query rows that share a kv head (the head group of one token, or of
// a few) against 16 keys a step, on mma.m16n8k16. Bound by HBM: the arithmetic
// is 8 heads deep at most, so the tensor cores only keep it off the FMA pipe;
// every key row is read once, straight into registers in fragment order:
//   scores   the contraction runs over features, whose order is free: lane
//            (g, c) = (lane / 4, lane % 4) holds the 16 bytes of features
//            32 u + 8 c of key g, which are the B fragments of two k-steps;
//   values   lane (g, c) holds features 64 w + 8 g .. + 7 of keys 2c, 2c + 1,
//            2c + 8, 2c + 9; the column order is free too, so the pairs of one
//            feature of two keys are one byte permute away from B fragments.
// A warp owns a run of steps with its own running maximum; warps and the CTAs
// of a cluster merge at the end through (distributed) shared memory, in a
// fixed order. Weights enter the value product as two bf16 terms (high and
// low half), which costs idle tensor time and keeps them to 2^-17.
constexpr int FR_MAXCL = 16;

template <int NU, int ROWS, int W>
__global__ void __launch_bounds__(W * 32) attend_few_kernel(const __grid_constant__ AttnCall c) {
    constexpr int NW = (NU + 1) / 2, DP = NW * 64;
    extern __shared__ __align__(16) float fsm[];
    float *so = fsm;                               // [W][ROWS][DP]
    float *sm = so + W * ROWS * DP;                // [W][ROWS] maxima
    float *sl = sm + W * ROWS;                     // [W][ROWS] sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
    const int rank = blockIdx.x, ncta = gridDim.x;   // the cluster spans x
    const int head = blockIdx.y % c.hkv, tile = blockIdx.y / c.hkv, seq = blockIdx.z;
    const int rows_total = c.lens ? c.rep : c.n * c.rep, r0 = tile * ROWS, nrows = min(ROWS, rows_total - r0);
    auto token_of = [&](int r) { return c.lens ? seq : (r0 + r) / c.rep; };
    auto qhead_of = [&](int r) { return head * c.rep + (r0 + r) % c.rep; };
    if (c.lens && c.lens[seq] < 0) return;         // a finished sequence: the whole cluster

    // the item's keys
    const int pmin = query_pos(c, token_of(0)), pmax = query_pos(c, token_of(nrows - 1));
    Span sp;
    const uint16_t *kb, *vb;
    if (c.lens) {
        const int lo = window_lo(c, pmax);
        sp.a1 = max(0, min(c.sinks, lo) - c.prefix);
        sp.c0 = sp.c1 = 0;
        sp.b0 = max(0, lo - c.prefix);
        sp.b1 = pmax + 1 - c.prefix;
        const size_t o = ((size_t)seq * c.hkv + head) * c.tcap * c.D;
        kb = c.tk + o;
        vb = c.tv + o;
    } else {
        sp = span_of(c, window_lo(c, pmin), pmax + 1);
        kb = c.k + (size_t)head * c.cap * c.D;
        vb = c.v + (size_t)head * c.cap * c.D;
    }
    const int na = (sp.a1 + 15) / 16, nc = (max(0, sp.c1 - sp.c0) + 15) / 16, nb = (max(0, sp.b1 - sp.b0) + 15) / 16;
    const int ns = na + nc + nb, wg = rank * W + warp, nwg = ncta * W;
    const int st0 = (int)((int64_t)ns * wg / nwg), st1 = (int)((int64_t)ns * (wg + 1) / nwg);

    // query fragments: rows g and g + 8, features in the keys' order
    uint32_t qa[NU][ROWS > 8 ? 8 : 4];
#pragma unroll
    for (int u = 0; u < NU; u++)
#pragma unroll
        for (int hf = 0; hf < (ROWS > 8 ? 2 : 1); hf++) {
            const int r = g + 8 * hf, f = 32 * u + 8 * cc;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < nrows && f < c.D)
                v = *reinterpret_cast<const uint4 *>(c.q + token_of(r) * c.q_stride + (int64_t)qhead_of(r) * c.D + f);
            qa[u][4 * hf] = v.x;
            qa[u][4 * hf + 1] = v.y;
            qa[u][4 * hf + 2] = v.z;
            qa[u][4 * hf + 3] = v.w;
        }
    const bool multi = pmin != pmax;               // rows at several positions: masks per row
    const int p0 = multi && g < nrows ? query_pos(c, token_of(g)) : pmax;
    const int p1 = multi && g + 8 < nrows ? query_pos(c, token_of(g + 8)) : pmax;
    const float s2 = c.scale * LOG2E;

    float o[NW * 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < NW * 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    auto step_slots = [&](int st, int &s, int &e) {
        if (st < na) {
            s = 16 * st;
            e = sp.a1;
        } else if (st < na + nc) {
            s = sp.c0 + 16 * (st - na);
            e = sp.c1;
        } else {
            s = sp.b0 + 16 * (st - na - nc);
            e = sp.b1;
        }
    };
    uint4 kr[NU][2], vr[NW][4];
    auto load_k = [&](int st) {
        int s, e;
        step_slots(st, s, e);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            // past the end: the last row again, its score masked
            const uint16_t *row = kb + (size_t)min(s + 8 * t + g, e - 1) * c.D + 8 * cc;
#pragma unroll
            for (int u = 0; u < NU; u++) kr[u][t] = 32 * u + 8 * cc < c.D ? ldg_nc_v4(row + 32 * u) : make_uint4(0, 0, 0, 0);
        }
    };
    auto load_v = [&](int st) {
        int s, e;
        step_slots(st, s, e);
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const uint16_t *row = vb + (size_t)min(s + 2 * cc + (t & 1) + 8 * (t >> 1), e - 1) * c.D + 8 * g;
#pragma unroll
            for (int w = 0; w < NW; w++) vr[w][t] = 64 * w + 8 * g < c.D ? ldg_nc_v4(row + 64 * w) : make_uint4(0, 0, 0, 0);
        }
    };
    if (st0 < st1) {
        load_k(st0);
        load_v(st0);
    }
    for (int st = st0; st < st1; st++) {
        float z[2][4];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            z[t][0] = z[t][1] = z[t][2] = z[t][3] = 0.f;
#pragma unroll
            for (int u = 0; u < NU; u++) {
                uint32_t a0[4] = {qa[u][0], ROWS > 8 ? qa[u][ROWS > 8 ? 4 : 0] : 0u, qa[u][1],
                                  ROWS > 8 ? qa[u][ROWS > 8 ? 5 : 0] : 0u};
                uint32_t a1[4] = {qa[u][2], ROWS > 8 ? qa[u][ROWS > 8 ? 6 : 0] : 0u, qa[u][3],
                                  ROWS > 8 ? qa[u][ROWS > 8 ? 7 : 0] : 0u};
                mma_bf16_16816(z[t], a0, kr[u][t].x, kr[u][t].y);
                mma_bf16_16816(z[t], a1, kr[u][t].z, kr[u][t].w);
            }
        }
        if (st + 1 < st1) load_k(st + 1);
        int s, e;
        step_slots(st, s, e);
        if (s + 16 > e || multi) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int key = s + 8 * t + 2 * cc + x;
                    bool see0 = key < e, see1 = see0;
                    if (multi) {
                        const int kp = slot_pos(c, key);
                        see0 = see0 && kp <= p0 && (kp >= window_lo(c, p0) || kp < c.sinks);
                        see1 = see1 && kp <= p1 && (kp >= window_lo(c, p1) || kp < c.sinks);
                    }
                    if (!see0) z[t][x] = -INFINITY;
                    if (!see1) z[t][2 + x] = -INFINITY;
                }
        }
        uint32_t ph[4], pl[4];
        auto half = [&](int x, float &m, float &l) {
            float mx = fmaxf(fmaxf(z[0][x], z[0][x + 1]), fmaxf(z[1][x], z[1][x + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn;
            if (__any_sync(0xffffffffu, mn > m)) {
                const float a = exp2f((m - mu) * s2);
                l *= a;
#pragma unroll
                for (int j = 0; j < NW * 8; j++) {
                    o[j][x] *= a;
                    o[j][x + 1] *= a;
                }
                m = mn;
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const float e0 = exp2f((z[t][x] - mu) * s2), e1 = exp2f((z[t][x + 1] - mu) * s2);
                l += e0 + e1;
                const uint32_t h = pack_bf2(e0, e1);
                ph[2 * t + x / 2] = h;
                pl[2 * t + x / 2] = pack_bf2(e0 - lo_bf(h), e1 - hi_bf(h));
            }
        };
        half(0, m0, l0);
        if constexpr (ROWS > 8) half(2, m1, l1);
        else ph[1] = ph[3] = pl[1] = pl[3] = 0u;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const uint32_t *y0 = &vr[w][0].x, *y1 = &vr[w][1].x, *y2 = &vr[w][2].x, *y3 = &vr[w][3].x;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
                const uint32_t b0 = __byte_perm(y0[j / 2], y1[j / 2], sel), b1 = __byte_perm(y2[j / 2], y3[j / 2], sel);
                mma_bf16_16816(o[8 * w + j], ph, b0, b1);
                mma_bf16_16816(o[8 * w + j], pl, b0, b1);
            }
        }
        if (st + 1 < st1) load_v(st + 1);
    }

    // row sums over the quad, then this warp's result to shared memory
#pragma unroll
    for (int hf = 0; hf < (ROWS > 8 ? 2 : 1); hf++) {
        float l = hf ? l1 : l0;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        const int r = g + 8 * hf;
        if (cc == 0) {
            sm[warp * ROWS + r] = hf ? m1 : m0;
            sl[warp * ROWS + r] = l;
        }
        // columns 2 cc and 2 cc + 1 of tile j are features 64 w + 16 cc + j and + 8 + j
        float *dst = so + (size_t)(warp * ROWS + r) * DP;
#pragma unroll
        for (int w = 0; w < NW; w++)
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *reinterpret_cast<float4 *>(dst + 64 * w + 16 * cc + 8 * x + j) =
                        make_float4(o[8 * w + j][2 * hf + x], o[8 * w + j + 1][2 * hf + x],
                                    o[8 * w + j + 2][2 * hf + x], o[8 * w + j + 3][2 * hf + x]);
    }
    __syncthreads();
    // the CTA's warps into warp 0's rows
    for (int i = tid; i < nrows * (DP / 4); i += W * 32) {
        const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, sm[w * ROWS + r]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY)
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float a = exp2f((sm[w * ROWS + r] - M) * s2);
                const float4 v = *reinterpret_cast<const float4 *>(so + (size_t)(w * ROWS + r) * DP + d);
                acc.x = fmaf(a, v.x, acc.x);
                acc.y = fmaf(a, v.y, acc.y);
                acc.z = fmaf(a, v.z, acc.z);
                acc.w = fmaf(a, v.w, acc.w);
            }
        *reinterpret_cast<float4 *>(so + (size_t)r * DP + d) = acc;
    }
    __syncthreads();
    if (tid < nrows) {
        float M = -INFINITY, L = 0.f;
        for (int w = 0; w < W; w++) M = fmaxf(M, sm[w * ROWS + tid]);
        if (M != -INFINITY)
            for (int w = 0; w < W; w++) L += sl[w * ROWS + tid] * exp2f((sm[w * ROWS + tid] - M) * s2);
        sm[tid] = M;
        sl[tid] = L;
    }
    cluster_sync_all();
    pdl_wait();                                    // the prefix half's results
    // rows x features over the cluster's CTAs: ranks in order, then the prefix's splits
    for (int i = rank * W * 32 + tid; i < nrows * (c.D / 4); i += ncta * W * 32) {
        const int r = i / (c.D / 4), d = 4 * (i % (c.D / 4)), token = token_of(r), qh = qhead_of(r);
        float M = -INFINITY;
        for (int k = 0; k < ncta; k++) M = fmaxf(M, ld_cluster(sm + r, k));
        const int64_t row = (int64_t)token * c.hq + qh, prow = (int64_t)c.n * c.hq;
        for (int k = 0; k < c.parts; k++) M = fmaxf(M, c.part_ml[k * prow + row].x);
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (M != -INFINITY) {
            for (int k = 0; k < ncta; k++) {
                const float a = exp2f((ld_cluster(sm + r, k) - M) * s2);
                const float4 v = ld_cluster4(so + (size_t)r * DP + d, k);
                L = fmaf(a, ld_cluster(sl + r, k), L);
                acc.x = fmaf(a, v.x, acc.x);
                acc.y = fmaf(a, v.y, acc.y);
                acc.z = fmaf(a, v.z, acc.z);
                acc.w = fmaf(a, v.w, acc.w);
            }
            for (int k = 0; k < c.parts; k++) {
                const float2 ml = c.part_ml[k * prow + row];
                const float a = exp2f((ml.x - M) * s2);
                if (ml.x == -INFINITY) continue;
                const float4 v = *reinterpret_cast<const float4 *>(c.part_o + (k * prow + row) * c.D + d);
                L = fmaf(a, ml.y, L);
                acc.x = fmaf(a, v.x, acc.x);
                acc.y = fmaf(a, v.y, acc.y);
                acc.z = fmaf(a, v.z, acc.z);
                acc.w = fmaf(a, v.w, acc.w);
            }
        }
        const float inv = M == -INFINITY ? 0.f : 1.0f / L;   // a row that sees nothing is zero
        *reinterpret_cast<uint2 *>(c.out + token * c.out_stride + (int64_t)qh * c.D + d) =
            make_uint2(pack_bf2(acc.x * inv, acc.y * inv), pack_bf2(acc.z * inv, acc.w * inv));
    }
    cluster_sync_all();                            // no CTA leaves while its shared memory is read
}

template <int NU, int ROWS, int W>
static int launch_few(const AttnCall &c, int cl, int tiles, bool pdl, cudaStream_t st) {
    constexpr int DP = (NU + 1) / 2 * 64;
    auto kern = attend_few_kernel<NU, ROWS, W>;
    const size_t smem = (size_t)W * ROWS * (DP + 2) * 4;
    if (!smem_allowed((const void *)kern, smem) || (cl > 8 && !nonportable_allowed((const void *)kern))) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cl, c.hkv * tiles, c.lens ? c.n : 1);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    MLXD_CHECK(cudaLaunchKernelEx(&cfg, kern, c));
    return 0;
}

// rows: query rows of an item that share a kv head; keys: the most that an
// item reads
static int attend_few(const AttnCall &c, int rows, int keys, bool pdl, cudaStream_t st) {
    const int R = rows > 8 ? 16 : 8, tiles = (rows + R - 1) / R;
    if ((int64_t)c.hkv * tiles > 65535 || (c.lens && c.n > 65535)) {
        set_error("attention: too many rows for one launch");
        return -1;
    }
    const int64_t items = (int64_t)c.hkv * tiles * (c.lens ? c.n : 1);
    // fill the SMs while every warp of 8 still has a step of 16 keys
    int cl = 1;
    while (cl < FR_MAXCL && items * cl * 2 <= num_sms() && keys > cl * 8 * 16) cl *= 2;
    const int nu = (c.D + 31) / 32;
    switch (nu * 2 + (R > 8)) {
    case 2: return launch_few<1, 8, 8>(c, cl, tiles, pdl, st);
    case 3: return launch_few<1, 16, 8>(c, cl, tiles, pdl, st);
    case 4: return launch_few<2, 8, 8>(c, cl, tiles, pdl, st);
    case 5: return launch_few<2, 16, 8>(c, cl, tiles, pdl, st);
    case 6: return launch_few<3, 8, 8>(c, cl, tiles, pdl, st);
    case 7: return launch_few<3, 16, 8>(c, cl, tiles, pdl, st);
    case 8: return launch_few<4, 8, 8>(c, cl, tiles, pdl, st);
    case 9: return launch_few<4, 16, 8>(c, cl, tiles, pdl, st);
    }
    set_error("attention: head dim %d", c.D);
    return -1;
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
    if (c.D <= 128 && !c.lens && (c.n == 1 || c.n * c.rep <= 16)) {
        const int last = c.pos0 + c.n;
        const int keys = c.window && (int64_t)c.window + c.n - 1 + c.sinks < last ? c.window + c.n - 1 + c.sinks : last;
        return attend_few(c, c.n * c.rep, keys, false, st);
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
    c.total = total;
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
    c.prefix = c.total = g->prefix_len;
    return attend(c, ws, ws_bytes, (cudaStream_t)stream);
}

}  // extern "C"
