// Token scores: for each row of logits x the log probability of a given token,
// the entropy and the most likely tokens.
//
//   M = max x,  S = sum_{i != argmax} e^(x_i - M),  W = sum (x_i - M) e^(x_i - M)
//   logprob(t) = x_t - M - log1p(S),   H = log1p(S) - W / (1 + S)
//
// Bound by HBM: one pass reads every logit once. A thread keeps its largest
// logit out of its own sums (so that a peaked row keeps its small terms), the
// sums relative to a reference that moves only when the maximum has grown by
// more than e^5. Merging thread, warp, CTA and cluster results rescales to the
// common maximum and lets every held-out logit but the row's join.
//
// Top list: the k-th largest of the maxima of thread groups is a lower bound
// T of the k-th largest logit, and no group below T holds any of the k; so
// only k groups' logits (of 64) are read again, from L2, and what reaches T is
// ranked by counting. Keys (value, index) are distinct, ties cost nothing.
#include "common.cuh"
#include "kernels.h"

namespace mlxd {

constexpr int SC_THREADS = 256, SC_GROUPS = SC_THREADS / 4, SC_TOP = 32, SC_CAND = 1024, SC_MAXCL = 16;
constexpr int SC_UNROLL = 4;

struct ScoreCall {
    const void *x;
    int64_t stride;
    int rows, V, top;
    const int32_t *targets;
    float *lp, *ent, *tlp;
    int32_t *ids;
};

typedef unsigned long long u64;

// order of the top list: larger logits first, equal values (+0 and -0 too) by
// index; never NaN
MLXD_DEV u64 sc_key(float v, int i) {
    const uint32_t u = __float_as_uint(v + 0.0f);
    return ((u64)((u & 0x80000000u) ? ~u : (u | 0x80000000u)) << 32) | (uint32_t)~i;
}
MLXD_DEV float sc_val(u64 key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
MLXD_DEV int sc_idx(u64 key) { return (int)~(uint32_t)key; }
MLXD_DEV float sc_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
MLXD_DEV float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

template <typename T>
MLXD_DEV float sc_load(const T *p, int i);
template <>
MLXD_DEV float sc_load<uint16_t>(const uint16_t *p, int i) { return bf2f(p[i]); }
template <>
MLXD_DEV float sc_load<float>(const float *p, int i) { return p[i]; }
// the logits of a 16-byte vector
MLXD_DEV void sc_unpack(const uint4 &v, float (&x)[8]) {
    x[0] = lo_bf(v.x); x[1] = hi_bf(v.x); x[2] = lo_bf(v.y); x[3] = hi_bf(v.y);
    x[4] = lo_bf(v.z); x[5] = hi_bf(v.z); x[6] = lo_bf(v.w); x[7] = hi_bf(v.w);
}
MLXD_DEV void sc_unpack(const uint4 &v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
}

constexpr float SC_LOG2E = 1.4426950408889634f, SC_LN2 = 0.6931471805599453f;

// sums over what was seen but its largest logit: s of 2^z and w of z 2^z, z =
// (x - ref) log2 e; best/at: the held-out logit (-inf: none above -inf yet)
struct ScoreSums {
    float ref, s, w, best;
    int at;
};

template <int N>
MLXD_DEV void sc_add(ScoreSums &a, float (&x)[N], int base) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < N; i++) mx = fmaxf(mx, x[i]);
    if (mx > a.best) {
        int j = N - 1;
#pragma unroll
        for (int i = N - 2; i >= 0; i--) j = x[i] == mx ? i : j;
        const bool first = a.best == -INFINITY;
        if (first || mx > a.ref + 5.0f) {
            const float d = first ? 0.f : (a.ref - mx) * SC_LOG2E, f = sc_ex2(d);
            a.w = f * fmaf(d, a.s, a.w);
            a.s *= f;
            a.ref = mx;
        }
        if (!first) {                                // the old largest joins the sums
            const float z = fmaxf((a.best - a.ref) * SC_LOG2E, -200.f), e = sc_ex2(z);
            a.s += e;
            a.w = fmaf(z, e, a.w);
        }
        a.best = mx;
        a.at = base + j;
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = i == j ? -INFINITY : x[i];
    }
    // -inf counts 2^-200 = 0; NaN stays NaN
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float z = max_nan((x[i] - a.ref) * SC_LOG2E, -200.f), e = sc_ex2(z);
        a.s += e;
        a.w = fmaf(z, e, a.w);
    }
}

// (s, w) relative to ref, expressed relative to m >= ref's row maximum
MLXD_DEV void sc_move(float &s, float &w, float ref, float m) {
    const float d = fmaxf((ref - m) * SC_LOG2E, -200.f), f = sc_ex2(d);
    w = f * fmaf(d, s, w);
    s *= f;
}
// the held-out logit v joins sums relative to m
MLXD_DEV void sc_join(float &s, float &w, float v, float m) {
    const float z = fmaxf((v - m) * SC_LOG2E, -200.f), e = sc_ex2(z);
    s += e;
    w = fmaf(z, e, w);
}

// a CTA's part of a row
struct ScorePart {
    u64 key;                   // its largest logit (0: none above -inf)
    float s, w;                // the rest, relative to that
    int count;                 // entries of list
    u64 list[SC_TOP];          // its largest logits above -inf, descending
};

MLXD_DEV u64 ld_cluster64(const u64 *p, int rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(cluster_addr(p, rank)));
    return v;
}

template <typename T>
__global__ void __launch_bounds__(SC_THREADS, 4) scores_kernel(const __grid_constant__ ScoreCall c) {
    constexpr int N = 16 / sizeof(T), NWARP = SC_THREADS / 32;
    __shared__ ScorePart part;
    __shared__ u64 s_wkey[NWARP], s_gkey[SC_GROUPS], s_cand[SC_CAND], s_t;
    __shared__ float s_ws[NWARP][2];
    __shared__ int s_flag[SC_GROUPS], s_nflag, s_ncand;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x, ncta = gridDim.x;   // the cluster spans x
    const int64_t row = blockIdx.y + (int64_t)blockIdx.z * 65535;
    if (row >= c.rows) return;                       // the whole cluster
    const T *x = (const T *)c.x + row * c.stride;
    // 16-byte vectors of the row, and up to N - 1 logits before and after them (CTA 0)
    const int skew = (int)(((uintptr_t)x & 15) / sizeof(T)), head = min(skew ? N - skew : 0, c.V);
    const int nvec = (c.V - head) / N, tail0 = head + nvec * N;
    const int v0 = (int)((int64_t)nvec * rank / ncta), v1 = (int)((int64_t)nvec * (rank + 1) / ncta);
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
    const int extras = rank == 0 ? head + c.V - tail0 : 0;
    auto extra_at = [&](int i) { return i < head ? i : tail0 + i - head; };

    ScoreSums a = {0.f, 0.f, 0.f, -INFINITY, 0};
    // in index order, so that a thread holds out the first of equal logits
    if (tid < min(head, extras)) {
        float e[1] = {sc_load(x, tid)};
        sc_add<1>(a, e, tid);
    }
    for (int v = v0 + tid; v < v1; v += SC_UNROLL * SC_THREADS) {
        uint4 u[SC_UNROLL];
#pragma unroll
        for (int k = 0; k < SC_UNROLL; k++)
            if (v + k * SC_THREADS < v1) u[k] = ldg_nc_v4(xv + v + k * SC_THREADS);
#pragma unroll
        for (int k = 0; k < SC_UNROLL; k++)
            if (v + k * SC_THREADS < v1) {
                float e[N];
                sc_unpack(u[k], e);
                sc_add<N>(a, e, head + (v + k * SC_THREADS) * N);
            }
    }
    if (tid >= head && tid < extras) {
        float e[1] = {sc_load(x, extra_at(tid))};
        sc_add<1>(a, e, extra_at(tid));
    }

    // the CTA's largest logit and the sums of the rest
    const u64 mine = a.best > -INFINITY ? sc_key(a.best, a.at) : 0ull;
    u64 k1 = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, k1, o);
        k1 = other > k1 ? other : k1;
        if (o == 2 && (lane & 3) == 0) s_gkey[tid >> 2] = k1;
    }
    if (lane == 0) s_wkey[warp] = k1;
    if (tid == 0) s_nflag = s_ncand = 0;
    __syncthreads();
    u64 key = s_wkey[0];
#pragma unroll
    for (int w = 1; w < NWARP; w++) key = s_wkey[w] > key ? s_wkey[w] : key;
    const float m = key ? sc_val(key) : -INFINITY;
    if (a.best > -INFINITY) {
        sc_move(a.s, a.w, a.ref, m);
        if (mine != key) sc_join(a.s, a.w, a.best, m);
    }
    a.s = warp_sum(a.s);
    a.w = warp_sum(a.w);
    if (lane == 0) {
        s_ws[warp][0] = a.s;
        s_ws[warp][1] = a.w;
    }
    // T: the top-th largest group maximum (all above -inf when there are fewer)
    if (c.top && tid < SC_GROUPS) {
        const u64 g = s_gkey[tid];
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < SC_GROUPS; i++) above += s_gkey[i] > g;
        if (g && above < c.top) s_flag[atomicAdd(&s_nflag, 1)] = tid;
        if (g && above == c.top - 1) s_t = g;
    }
    __syncthreads();
    if (tid == 0) {
        float s = 0.f, w = 0.f;
        for (int i = 0; i < NWARP; i++) {
            s += s_ws[i][0];
            w += s_ws[i][1];
        }
        part.key = key;
        part.s = s;
        part.w = w;
    }
    if (c.top) {
        const int nflag = s_nflag;
        const u64 T0 = nflag == c.top ? s_t : 1ull;
        const float tv = nflag == c.top ? sc_val(T0) : -INFINITY;
        auto offer = [&](float v, int i) {
            if (v >= tv && v > -INFINITY) {
                const u64 k = sc_key(v, i);
                if (k >= T0) {
                    const int at = atomicAdd(&s_ncand, 1);
                    if (at < SC_CAND) s_cand[at] = k;
                }
            }
        };
        for (int f = warp; f < nflag; f += NWARP) {
            const int g = s_flag[f];
            for (int i = lane;; i += 32) {
                const int v = v0 + 4 * g + (i & 3) + (i >> 2) * SC_THREADS;
                if (v - (i & 3) >= v1) break;
                if (v >= v1) continue;
                float e[N];
                sc_unpack(ldg_nc_v4(xv + v), e);
#pragma unroll
                for (int j = 0; j < N; j++) offer(e[j], head + v * N + j);
            }
            if (lane < 4 && 4 * g + lane < extras) offer(sc_load(x, extra_at(4 * g + lane)), extra_at(4 * g + lane));
        }
        __syncthreads();
        const int nc = s_ncand;
        if (nc <= SC_CAND) {
            for (int i = tid; i < nc; i += SC_THREADS) {
                const u64 k = s_cand[i];
                int above = 0;
                for (int j = 0; j < nc; j++) above += s_cand[j] > k;
                if (above < c.top) part.list[above] = k;
            }
            if (tid == 0) part.count = min(nc, c.top);
        } else {
            // more reach T than there is room for (k groups that hold nearly all of the largest): the
            // largest below the last one, again and again
            u64 last = ~0ull;
            for (int r = 0; r < c.top; r++) {
                u64 b = 0;
                auto look = [&](float v, int i) {
                    if (v > -INFINITY) {
                        const u64 k = sc_key(v, i);
                        b = k < last && k > b ? k : b;
                    }
                };
                if (tid < extras) look(sc_load(x, extra_at(tid)), extra_at(tid));
                for (int v = v0 + tid; v < v1; v += SC_THREADS) {
                    float e[N];
                    sc_unpack(ldg_nc_v4(xv + v), e);
#pragma unroll
                    for (int j = 0; j < N; j++) look(e[j], head + v * N + j);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) {
                    const u64 other = __shfl_xor_sync(0xffffffffu, b, o);
                    b = other > b ? other : b;
                }
                __syncthreads();
                if (lane == 0) s_wkey[warp] = b;
                __syncthreads();
                last = 0;
                for (int w = 0; w < NWARP; w++) last = s_wkey[w] > last ? s_wkey[w] : last;
                if (tid == 0) part.list[r] = last;
            }
            if (tid == 0) part.count = c.top;
        }
    }
    if (ncta > 1) {
        cluster_sync_all();
        if (rank != 0) {
            cluster_sync_all();                      // until CTA 0 has read this one's part
            return;
        }
    } else {
        __syncthreads();
    }

    // CTA 0: the row from its parts
    __shared__ u64 s_list[SC_TOP];
    __shared__ float s_m, s_ls, s_ent;
    __shared__ int s_count;
    if (warp == 0) {
        u64 pk = 0;
        float s = 0.f, w = 0.f;
        if (lane < ncta) {
            pk = ld_cluster64(&part.key, lane);
            s = ld_cluster(&part.s, lane);
            w = ld_cluster(&part.w, lane);
        }
        u64 best = pk;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
        }
        const float M = best ? sc_val(best) : -INFINITY;
        if (pk) {
            sc_move(s, w, sc_val(pk), M);
            if (pk != best) sc_join(s, w, sc_val(pk), M);
        }
        s = warp_sum(s);
        w = warp_sum(w);
        if (lane == 0) {
            const float ls = M < INFINITY ? log1pf(s) : __int_as_float(0x7fc00000);   // +inf has no scores
            const bool empty = !best && s == 0.f;    // nothing above -inf and no NaN
            s_m = M;
            s_ls = ls;
            s_ent = empty ? 0.f : ls - w * SC_LN2 / (1.f + s);
            s_count = 0;
        }
    }
    if (c.top && ncta > 1) {
        for (int i = tid; i < ncta * c.top; i += SC_THREADS) {
            const int k = i / c.top, j = i - k * c.top;
            int n = (int)__float_as_uint(ld_cluster(reinterpret_cast<const float *>(&part.count), k));
            s_cand[i] = j < n ? ld_cluster64(&part.list[j], k) : 0ull;
        }
    }
    __syncthreads();
    if (ncta > 1) cluster_sync_all();
    const float M = s_m, ls = s_ls;
    const bool empty = M == -INFINITY && !isnan(ls);
    if (tid == 0) {
        if (c.lp) {
            const int t = c.targets[row];
            c.lp[row] = t < 0 || t >= c.V ? __int_as_float(0x7fc00000) : empty ? -INFINITY : sc_load(x, t) - M - ls;
        }
        if (c.ent) c.ent[row] = s_ent;
    }
    if (!c.top) return;
    if (ncta > 1) {
        for (int i = tid; i < ncta * c.top; i += SC_THREADS) {
            const u64 k = s_cand[i];
            int above = 0;
            for (int j = 0; j < ncta * c.top; j++) above += s_cand[j] > k;
            if (k && above < c.top) {
                s_list[above] = k;
                atomicAdd(&s_count, 1);
            }
        }
    } else {
        if (tid < part.count) s_list[tid] = part.list[tid];
        if (tid == 0) s_count = part.count;
    }
    __syncthreads();
    int count = s_count;
    if (tid < count) {
        const u64 k = s_list[tid];
        if (c.ids) c.ids[row * c.top + tid] = sc_idx(k);
        if (c.tlp) c.tlp[row * c.top + tid] = sc_val(k) - M - ls;
    }
    // fewer than top logits above -inf: the first ones at -inf, then the first NaNs
    for (int kind = 0; kind < 2 && count < c.top; kind++)
        for (int i0 = 0; i0 < c.V && count < c.top; i0 += SC_THREADS) {
            const float v = i0 + tid < c.V ? sc_load(x, i0 + tid) : 0.f;
            const bool hit = kind ? isnan(v) : v == -INFINITY;
            const unsigned b = __ballot_sync(0xffffffffu, hit);
            __syncthreads();
            if (lane == 0) s_flag[warp] = __popc(b);
            __syncthreads();
            int at = count + __popc(b & ((1u << lane) - 1u));
            for (int w = 0; w < NWARP; w++) {
                if (w < warp) at += s_flag[w];
                count += s_flag[w];
            }
            if (hit && at < c.top) {
                if (c.ids) c.ids[row * c.top + at] = i0 + tid;
                if (c.tlp) c.tlp[row * c.top + at] = isnan(ls) ? ls : kind ? v : -INFINITY;
            }
        }
}

template <typename T>
static int launch_scores(const ScoreCall &c, cudaStream_t st) {
    auto kern = scores_kernel<T>;
    // few rows: a cluster per row while there are SMs and every thread keeps a vector
    int cl = 1;
    while (cl < SC_MAXCL && (int64_t)c.rows * cl * 2 <= num_sms() && c.V > cl * SC_THREADS * (int)(16 / sizeof(T))) cl *= 2;
    if (cl > 8 && !nonportable_allowed((const void *)kern)) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cl, c.rows < 65535 ? c.rows : 65535, (c.rows + 65534) / 65535);
    cfg.blockDim = dim3(SC_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cl;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    MLXD_CHECK(cudaLaunchKernelEx(&cfg, kern, c));
    return 0;
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
    if ((uintptr_t)logits % (dtype == MLXD_BF16 ? 2 : 4)) {
        set_error("token_scores: misaligned logits");
        return -1;
    }
    if (rows == 0) return 0;
    if (!on_device(logits, "token_scores: logits") || (targets && !on_device(targets, "token_scores: targets")) ||
        (logprobs && !on_device(logprobs, "token_scores: logprobs")) ||
        (entropy && !on_device(entropy, "token_scores: entropy")) ||
        (n_top && top_ids && !on_device(top_ids, "token_scores: top ids")) ||
        (n_top && top_logprobs && !on_device(top_logprobs, "token_scores: top logprobs")))
        return -1;
    const ScoreCall c = {logits, row_stride, rows, V, n_top, targets, logprobs, entropy, top_logprobs, top_ids};
    return dtype == MLXD_BF16 ? launch_scores<uint16_t>(c, (cudaStream_t)stream)
                              : launch_scores<float>(c, (cudaStream_t)stream);
}
