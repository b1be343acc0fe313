// Token scores: for each row of logits x the log probability of a given token,
// the entropy and the most likely tokens.
//
//   M = max x,  S = sum_{i != argmax} e^(x_i - M),  W = sum (x_i - M) e^(x_i - M)
//   logprob(t) = x_t - M - log1p(S),   H = log1p(S) - W / (1 + S)
//
// Bound by HBM: one pass reads every logit once (the first part of it twice,
// the second time from L2), and the arithmetic, an exponential and some seven
// other instructions a logit, has to stay below the issue rate. T, the k-th
// largest of the maxima of 64 thread groups over the first part of a CTA's
// logits, bounds its k-th largest logit from below. A logit that reaches T goes
// to a list in shared memory (for random orders some 4 k of them); all others
// are summed relative to the first part's maximum, which they cannot exceed. At
// the end the list is ranked by counting (keys of value and index are distinct,
// ties cost nothing), and the listed logits but the largest join the sums in that
// order (a peaked row keeps its small terms; the threads' timing changes no bit).
// A row whose list overflows (rising or strided rows, thousands of ties) is read
// again with every thread's largest logit held out of its sums, and the list is
// made from the whole row's group maxima. Measured, 512 rows of 151936 bf16 with
// 20 alternatives: 50 us, 48% of the measured copy rate; 37 of them without the
// sums, the rest of the distance the selection's serial steps at a row's end.
// The same rows in f32: 67 us, 71%; 128 of them 49 us, 24% (fewer CTAs than SMs).
#include "common.cuh"
#include "kernels.h"

namespace mlxd {

constexpr int SC_THREADS = 256, SC_GROUPS = SC_THREADS / 4, SC_TOP = 32, SC_CAND = 1024, SC_MAXCL = 16;
constexpr int SC_MAXV = INT32_MAX - SC_THREADS;      // a step of the CTA past the end is still an int
// the first part: a quarter (a third 50.5, a sixth 53, an eighth 58 us: a looser T lists more)
constexpr int SC_UNROLL = 4, SC_PART = 4;

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

// logits that do not exceed ref by much: -inf counts 2^-200 = 0, NaN stays NaN
template <int N>
MLXD_DEV void sc_sum(ScoreSums &a, const float (&x)[N]) {
    if constexpr (N == 1) {
        const float z = max_nan((x[0] - a.ref) * SC_LOG2E, -200.f), e = sc_ex2(z);
        a.s += e;
        a.w = fmaf(z, e, a.w);
    } else {
        const u64 ref2 = pair2(-a.ref, -a.ref), log2e2 = pair2(SC_LOG2E, SC_LOG2E);
        u64 s2 = pair2(a.s, 0.f), w2 = pair2(a.w, 0.f);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            float z0, z1;
            unpair2(mul2(add2(pair2(x[i], x[i + 1]), ref2), log2e2), z0, z1);
            z0 = max_nan(z0, -200.f);
            z1 = max_nan(z1, -200.f);
            const u64 e = pair2(sc_ex2(z0), sc_ex2(z1));
            s2 = add2(s2, e);
            w2 = fma2(pair2(z0, z1), e, w2);
        }
        float t;
        unpair2(s2, a.s, t);
        a.s += t;
        unpair2(w2, a.w, t);
        a.w += t;
    }
}

// any logits: a larger one than before is held out in place of the old
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
        if (first && a.s == 0.f) {
            a.ref = mx;
        } else if (mx > a.ref + 5.0f) {
            const float d = (a.ref - mx) * SC_LOG2E, f = sc_ex2(d);
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
    sc_sum<N>(a, x);
}

// (s, w) relative to ref, expressed relative to the maximum m >= ref
MLXD_DEV void sc_move(float &s, float &w, float ref, float m) {
    if (s == 0.f) return;                            // nothing yet, whatever ref was
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

// the largest logit of a vector (NaN aside)
template <typename T>
MLXD_DEV float sc_max(const uint4 &v) {
    if constexpr (sizeof(T) == 2) {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
        const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        return fmaxf(__low2float(m), __high2float(m));
    } else {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
}

template <typename T>
__global__ void __launch_bounds__(SC_THREADS, 4) scores_kernel(const __grid_constant__ ScoreCall c) {
    constexpr int N = 16 / sizeof(T), NWARP = SC_THREADS / 32;
    __shared__ ScorePart part;
    __shared__ u64 s_wkey[NWARP], s_gkey[SC_GROUPS], s_cand[SC_CAND], s_sort[SC_CAND], s_t;
    __shared__ float s_ws[NWARP][2];
    __shared__ int s_flag[SC_THREADS], s_nflag, s_ncand;
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
    const int want = max(c.top, 4);                  // T's rank

    auto warp_max64 = [&](u64 k) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, k, o);
            k = other > k ? other : k;
        }
        return k;
    };
    auto block_max64 = [&](u64 k) {                  // two barriers
        k = warp_max64(k);
        __syncthreads();
        if (lane == 0) s_wkey[warp] = k;
        __syncthreads();
        k = s_wkey[0];
#pragma unroll
        for (int w = 1; w < NWARP; w++) k = s_wkey[w] > k ? s_wkey[w] : k;
        return k;
    };
    // f(list[i], how many of list[0 .. n) are larger) for every i, a thread each
    auto ranks = [&](const u64 *list, int n, auto f) {
        for (int i = tid; i < n; i += SC_THREADS) {
            const u64 k = list[i];
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) above += list[j] > k;
            f(k, above);
        }
    };
    // T from the threads' largest keys: the `want`-th largest of the maxima of
    // 64 thread groups (1: fewer hold anything above -inf)
    auto threshold = [&](u64 mine) {
        u64 q = mine;
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, q, o);
            q = other > q ? other : q;
        }
        __syncthreads();
        if ((lane & 3) == 0) s_gkey[tid >> 2] = q;
        if (tid == 0) {
            s_t = 1ull;
            s_nflag = 0;
        }
        __syncthreads();
        ranks(s_gkey, SC_GROUPS, [&](u64 g, int above) {
            if (g && above == want - 1) s_t = g;
        });
        __syncthreads();
        return s_t;
    };
    // What reaches T = threshold(mine) into s_cand, mine the threads' largest
    // keys over the CTA's logits. The threads' own keys are flagged against T,
    // so that some `want` threads' logits are read again.
    auto collect = [&](u64 mine) {
        const u64 t = threshold(mine);
        if (mine >= t) s_flag[atomicAdd(&s_nflag, 1)] = tid;
        __syncthreads();
        auto offer = [&](float v, int i) {
            if (!(v > -INFINITY)) return;
            const u64 k = sc_key(v, i);
            if (k < t) return;
            const int at = atomicAdd(&s_ncand, 1);
            if (at < SC_CAND) s_cand[at] = k;
        };
        // (flagged thread, round) over all threads: the loads of a list go out together
        const int nflag = s_nflag, per = (v1 - v0 + SC_THREADS - 1) / SC_THREADS;
        for (int i = tid; i < nflag * per; i += SC_THREADS) {
            const int f = i / per, v = v0 + s_flag[f] + (i - f * per) * SC_THREADS;
            if (v >= v1) continue;
            float e[N];
            sc_unpack(ldg_nc_v4(xv + v), e);
#pragma unroll
            for (int j = 0; j < N; j++) offer(e[j], head + v * N + j);
        }
        if (mine >= t && tid < extras) offer(sc_load(x, extra_at(tid)), extra_at(tid));
        __syncthreads();
    };

    if (tid == 0) s_ncand = 0;
    const int target = tid == 0 && rank == 0 && c.lp ? c.targets[row] : -1;
    // maxima of the first part: T as a value, and the reference of the sums
    float top = -INFINITY;
    const int rounds = (v1 - v0 + SC_THREADS - 1) / SC_THREADS, va = min(v1, v0 + (rounds + SC_PART - 1) / SC_PART * SC_THREADS);
    if (tid < extras) top = fmaxf(top, sc_load(x, extra_at(tid)));
    for (int v = v0 + tid; v < va; v += SC_UNROLL * SC_THREADS) {
        uint4 u[SC_UNROLL];
#pragma unroll
        for (int k = 0; k < SC_UNROLL; k++)
            if (v + k * SC_THREADS < va) u[k] = ldg_nc_v4(xv + v + k * SC_THREADS);
#pragma unroll
        for (int k = 0; k < SC_UNROLL; k++)
            if (v + k * SC_THREADS < va) top = fmaxf(top, sc_max<T>(u[k]));
    }
    const float xt = target >= 0 && target < c.V ? sc_load(x, target) : 0.f;   // on its way until the end
    const u64 mine1 = top > -INFINITY ? sc_key(top, tid) : 0ull, t0 = threshold(mine1), first = block_max64(mine1);
    const float tv = t0 > 1 ? sc_val(t0) : -3.4028235e38f;

    // all: what reaches T is listed, the rest summed
    ScoreSums a = {first ? sc_val(first) : 0.f, 0.f, 0.f, -INFINITY, 0};
    auto add = [&](auto &e, bool reaches, int base) {
        constexpr int M = sizeof(e) / 4;
        if (reaches) {
            unsigned hit = 0;
#pragma unroll
            for (int j = 0; j < M; j++) hit |= e[j] >= tv ? 1u << j : 0u;
            int at = atomicAdd(&s_ncand, __popc(hit));
            if (at + __popc(hit) > SC_CAND) return;  // the row is summed again
#pragma unroll
            for (int j = 0; j < M; j++)
                if (hit >> j & 1) {
                    s_cand[at++] = sc_key(e[j], base + j);
                    e[j] = -INFINITY;
                }
        }
        sc_sum<M>(a, e);
    };
    if (tid < min(head, extras)) {
        float e[1] = {sc_load(x, tid)};
        add(e, e[0] >= tv, tid);
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
                add(e, sc_max<T>(u[k]) >= tv, head + (v + k * SC_THREADS) * N);
            }
    }
    if (tid >= head && tid < extras) {
        float e[1] = {sc_load(x, extra_at(tid))};
        add(e, e[0] >= tv, extra_at(tid));
    }
    __syncthreads();

    // The CTA's largest logit and the sums of the rest. The list's order depends
    // on the threads' timing, its ranks do not: they give the same bits every time.
    int n = s_ncand;
    auto sort = [&] {
        ranks(s_cand, n, [&](u64 k, int above) { s_sort[above] = k; });
        __syncthreads();
    };
    u64 key = 0;
    if (n <= SC_CAND) {
        sort();
        if (n) {
            key = s_sort[0];
            const float m = sc_val(key);
            sc_move(a.s, a.w, a.ref, m);
            for (int i = tid ? tid : SC_THREADS; i < n; i += SC_THREADS) sc_join(a.s, a.w, sc_val(s_sort[i]), m);
        }
    } else {
        // again, in index order (a thread holds out the first of equal logits), and the list from these maxima
        a.s = a.w = 0.f;
        if (tid < min(head, extras)) {
            float e[1] = {sc_load(x, tid)};
            sc_add<1>(a, e, tid);
        }
        for (int v = v0 + tid; v < v1; v += SC_THREADS) {
            float e[N];
            sc_unpack(ldg_nc_v4(xv + v), e);
            sc_add<N>(a, e, head + v * N);
        }
        if (tid >= head && tid < extras) {
            float e[1] = {sc_load(x, extra_at(tid))};
            sc_add<1>(a, e, extra_at(tid));
        }
        const u64 mine = a.best > -INFINITY ? sc_key(a.best, a.at) : 0ull;
        key = block_max64(mine);
        if (key) {
            const float m = sc_val(key);
            sc_move(a.s, a.w, a.ref, m);
            if (mine && mine != key) sc_join(a.s, a.w, a.best, m);
        }
        if (c.top) {
            if (tid == 0) s_ncand = 0;
            collect(mine);
            n = s_ncand;
            if (n <= SC_CAND) sort();
        }
    }
    a.s = warp_sum(a.s);
    a.w = warp_sum(a.w);
    if (lane == 0) {
        s_ws[warp][0] = a.s;
        s_ws[warp][1] = a.w;
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
        if (n <= SC_CAND) {
            if (tid < min(n, c.top)) part.list[tid] = s_sort[tid];
            if (tid == 0) part.count = min(n, c.top);
        } else {
            // every logit above -inf of this CTA, as a key, to f
            auto each = [&](auto f) {
                if (tid < extras) f(sc_load(x, extra_at(tid)), extra_at(tid));
                for (int v = v0 + tid; v < v1; v += SC_THREADS) {
                    float e[N];
                    sc_unpack(ldg_nc_v4(xv + v), e);
#pragma unroll
                    for (int j = 0; j < N; j++) f(e[j], head + v * N + j);
                }
            };
            // a few threads hold nearly all of the largest: the largest below the last one, again and again
            u64 last = ~0ull;
            for (int r = 0; r < c.top; r++) {
                u64 b = 0;
                each([&](float v, int i) {
                    const u64 k = v > -INFINITY ? sc_key(v, i) : 0ull;
                    if (k < last) b = max(b, k);
                });
                last = block_max64(b);
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
        }
    }
    // the parts' lists: what is above the last entry of a full one
    if (c.top && ncta > 1) {
        u64 full = 0;
        if (lane < ncta) {
            const int n = (int)__float_as_uint(ld_cluster(reinterpret_cast<const float *>(&part.count), lane));
            if (n == c.top) full = ld_cluster64(&part.list[n - 1], lane);
            if (warp == 0) s_flag[lane] = n;
        }
        full = warp_max64(full);
        if (tid == 0) s_ncand = 0;
        __syncthreads();
        for (int i = tid; i < ncta * SC_TOP; i += SC_THREADS) {
            const int k = i / SC_TOP, j = i % SC_TOP;
            if (j >= s_flag[k]) continue;
            const u64 v = ld_cluster64(&part.list[j], k);
            if (v >= full) s_cand[atomicAdd(&s_ncand, 1)] = v;
        }
    }
    __syncthreads();
    if (ncta > 1) cluster_sync_all();
    const float M = s_m, ls = s_ls;
    const bool empty = M == -INFINITY && !isnan(ls);
    if (tid == 0) {
        if (c.lp)
            c.lp[row] = target < 0 || target >= c.V ? __int_as_float(0x7fc00000) : empty ? -INFINITY : xt - M - ls;
        if (c.ent) c.ent[row] = s_ent;
    }
    if (!c.top) return;
    if (ncta > 1) {
        ranks(s_cand, s_ncand, [&](u64 k, int above) {
            if (above < c.top) s_list[above] = k;
        });
        if (tid == 0) s_count = min(s_ncand, c.top);
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
    while (cl < SC_MAXCL && (int64_t)c.rows * cl * 2 <= num_sms() && c.V > 4 * cl * SC_THREADS * (int)(16 / sizeof(T))) cl *= 2;
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
                                      int32_t *top_ids, float *top_logprobs, void *stream) try {
    if ((dtype != MLXD_BF16 && dtype != MLXD_F32) || rows < 0 || V <= 0 || V > SC_MAXV || row_stride < 0 ||
        n_top < 0 || n_top > SC_TOP || n_top > V) {
        set_error("token_scores: bad arguments (n_top: at most 32 and V; V: below 2^31 - 256)");
        return -1;
    }
    if (logprobs && !targets) {
        set_error("token_scores: logprobs without targets");
        return -1;
    }
    if (rows == 0) return 0;
    if (!on_device(logits, "token_scores: logits", dtype == MLXD_BF16 ? 2 : 4) ||
        (logprobs && !on_device(targets, "token_scores: targets", 4)) ||
        (logprobs && !on_device(logprobs, "token_scores: logprobs", 4)) ||
        (entropy && !on_device(entropy, "token_scores: entropy", 4)) ||
        (n_top && top_ids && !on_device(top_ids, "token_scores: top ids", 4)) ||
        (n_top && top_logprobs && !on_device(top_logprobs, "token_scores: top logprobs", 4)))
        return -1;
    const ScoreCall c = {logits, row_stride, rows, V, n_top, targets, logprobs, entropy, top_logprobs, top_ids};
    return dtype == MLXD_BF16 ? launch_scores<uint16_t>(c, (cudaStream_t)stream)
                              : launch_scores<float>(c, (cudaStream_t)stream);
} catch (...) {   // no exception leaves a C entry
    set_error("token_scores: out of host memory");
    return -1;
}
