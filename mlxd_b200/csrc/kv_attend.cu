// Attention over the rows of a cache layer, and of a batch that shares a
// prefix, for callers that drive layers themselves.
//
//   out_i = sum_j e^(s (q_i . k_j) - m_i) v_j / sum_j e^(s (q_i . k_j) - m_i)
//
// over the keys j <= p_i with p_i - j < window or j < sinks, in one pass over
// the keys with a running maximum m_i.
#include <limits.h>
#include <math.h>
#include <new>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tc.cuh"

namespace mlxd {

constexpr float LOG2E = 1.4426950408889634f;
MLXD_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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
__host__ MLXD_DEV int window_lo(const AttnCall &c, int p) { return c.window && p >= c.window ? p - c.window + 1 : 0; }

// The slots that hold positions [lo, hi) and the sinks below lo: [0, a1),
// [c0, c1) (the wrapped end of a ring) and [b0, b1), ascending. In a wrapped
// ring [lo, hi) lies above the kept sinks and spans at most the ring.
struct Span {
    int a1, c0, c1, b0, b1;
};
MLXD_DEV Span span_of(const AttnCall &c, int lo, int hi) {
    Span s;
    s.a1 = min(min(c.sinks, lo), c.total);
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

// the partial results' room in a workspace: 148 CTAs (a B200's SMs) of 256 rows,
// whatever the call (more rows than that go unsplit, or in batches)
constexpr int64_t AT_WS_ROWS = 148 * 256;
static size_t at_ws_bytes(int D) { return (size_t)AT_WS_ROWS * ((D + 7) / 8 * 8 * 4 + 8) + 256; }

static float2 *at_ws_ml(void *ws, int D) { return (float2 *)((char *)ws + (size_t)AT_WS_ROWS * D * 4); }

// ---- few query rows per kv head (single tokens, tails): key-split warps
//
// Up to 16 query rows that share a kv head (the head group of one token, or of
// a few) against 16 keys a step, on mma.m16n8k16 with the keys and then the
// features as its 16 rows and the query rows as its 8 columns (the other way
// round takes up to three times the MMAs, at 28 clocks each: 11.0 against 9.6 us
// for one token over 2192 positions). Every key row is read once; in fragment
// order:
//   scores   S^T = K Q^T: the contraction runs over features, whose order is
//            free: lane (g, c) = (lane / 4, lane % 4) holds the 16 bytes of
//            features 32 u + 8 c of keys g and g + 8, the A fragments of two
//            k-steps;
//   values   O^T = V^T P^T: lane (g, c) holds features 64 w + 8 g .. + 7 of keys
//            2c, 2c + 1, 2c + 8, 2c + 9; the row order is free too, so the
//            pairs of one feature of two keys are one byte permute away from A
//            fragments; P^T is a transposing move of the weights.
// A warp owns a run of steps with its own running maximum; warps and the CTAs
// of a cluster merge at the end through (distributed) shared memory, in a
// fixed order. Weights enter the value product as two bf16 terms (to 2^-17):
// with up to 4 rows the low terms fill the other 4 columns, with up to 8 they
// take a second MMA; with 16 rows (wide heads, groups of more than 8 heads over a
// tail) that would cost what HBM leaves, so there the weights are rounded to bf16
// and the row sum adds the rounded ones.
constexpr int FR_MAXCL = 8;                        // CTAs of a cluster (the portable size)
constexpr int FR_PARTS = 56, FR_SRC = 64;          // splits of a prefix, and those with a cluster's CTAs

struct FewCall {
    int tails;                 // an item is one sequence's tail, else up to ROWS query rows over the cache
    int cluster;               // grid x is a cluster whose results meet, else each CTA's is partial
    float *part_o;             // partial results [grid x][prow], or null: the whole result to out
    float2 *part_ml;
    int64_t prow;
};

// shared memory of a warp: its ring, later its results
constexpr int FR_DEPTH = 2;
__host__ __device__ constexpr int fr_warp_floats(int nu, int rows) {
    const int nw = (nu + 1) / 2, ring = FR_DEPTH * (2 * nu + 4 * nw) * 32 * 4, res = rows * nw * 64;
    return ring > res ? ring : res;
}
MLXD_DEV uint32_t transpose8(uint32_t v) {           // 8 x 8 bf16 across the warp
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int NU, int ROWS, int W>
__global__ void __launch_bounds__(W * 32)
    attend_few_kernel(const __grid_constant__ AttnCall c, const __grid_constant__ FewCall t) {
    constexpr int NW = (NU + 1) / 2, DP = NW * 64, NT = ROWS > 8 ? 2 : 1;
    constexpr bool LOW = ROWS <= 8;                  // the weights' low terms too
    extern __shared__ __align__(16) float fsm[];
    float *so = fsm;                               // [W][ROWS][DP], in the rings' place
    float *sm = so + W * fr_warp_floats(NU, ROWS);   // [W][ROWS] maxima
    float *sl = sm + W * ROWS;                     // [W][ROWS] sums
    float *sw = sl + W * ROWS;                     // [sources][ROWS] weights at the end
    float *srow = sw + FR_SRC * ROWS;              // [ROWS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, cc = lane & 3;
    const int rank = blockIdx.x, ncta = gridDim.x;   // the item's CTAs
    const int head = blockIdx.y % c.hkv, tile = blockIdx.y / c.hkv, seq = blockIdx.z;
    const int rows_total = t.tails ? c.rep : c.n * c.rep, r0 = tile * ROWS, nrows = min(ROWS, rows_total - r0);
    const bool one = t.tails || c.n == 1;            // the rows are heads of one token
    auto token_of = [&](int r) { return t.tails ? seq : one ? 0 : (r0 + r) / c.rep; };
    auto qhead_of = [&](int r) { return head * c.rep + (one ? r0 + r : (r0 + r) % c.rep); };
    pdl_trigger();                                 // the kernel that joins may be put in place
    if (t.tails && c.lens[seq] < 0) {              // a finished sequence: the whole cluster
        pdl_wait();                                // (no later kernel may overtake the prefix's)
        return;
    }

    // positions of the rows (lane r: row r; -1: not asked) and the item's keys
    const int rp = lane < nrows ? query_pos(c, token_of(lane)) : -1;
    const int pmax = __reduce_max_sync(0xffffffffu, rp);
    const int pmin = __reduce_min_sync(0xffffffffu, rp < 0 ? INT32_MAX : rp);
    const bool multi = __any_sync(0xffffffffu, lane < nrows && rp != pmax);   // masks per row
    Span sp = {0, 0, 0, 0, 0};
    const uint16_t *kb, *vb;
    if (t.tails) {
        const int lo = window_lo(c, pmax);
        sp.a1 = max(0, min(c.sinks, lo) - c.prefix);
        sp.b0 = max(0, lo - c.prefix);
        sp.b1 = pmax + 1 - c.prefix;
        const size_t o = ((size_t)seq * c.hkv + head) * c.tcap * c.D;
        kb = c.tk + o;
        vb = c.tv + o;
    } else {
        if (pmax >= 0) sp = span_of(c, window_lo(c, pmin), pmax + 1);
        kb = c.k + (size_t)head * c.cap * c.D;
        vb = c.v + (size_t)head * c.cap * c.D;
    }
    // (consecutive runs lie on different CTAs, so the longer ones do too)
    const int na = (sp.a1 + 15) / 16, nc = (max(0, sp.c1 - sp.c0) + 15) / 16, nb = (max(0, sp.b1 - sp.b0) + 15) / 16;
    const int ns = na + nc + nb, wg = warp * ncta + rank, nwg = ncta * W;
    const int each = ns / nwg, more = ns - each * nwg;   // the first `more` warps take one step more
    const int st0 = each * wg + min(wg, more), st1 = st0 + each + (wg < more);

    auto step_slots = [&](int st, int &s, int &e) {
        const bool a = st < na, b = st >= na + nc;
        s = a ? 16 * st : b ? sp.b0 + 16 * (st - na - nc) : sp.c0 + 16 * (st - na);
        e = a ? sp.a1 : b ? sp.b1 : sp.c1;
    };
    // A step's rows go through a ring of FR_DEPTH stages in shared memory, the warp's own: deep prefetch without
    // registers or CTA barriers.
    constexpr int KV = 2 * NU + 4 * NW;              // 16-byte pieces of a lane per step
    uint4 *ring = reinterpret_cast<uint4 *>(fsm) + (size_t)warp * FR_DEPTH * KV * 32 + lane;
    int put = 0, get = 0;                            // ring stages
    // The keys' pieces [16][4 NU] are copied in whole rows, so that an instruction meets 4 cache lines and not 8 (what
    // bounds the copies is the rate of lines: 131072 positions 115 -> 105 us, 32768 35.5 -> 33.4); odd rows swap
    // their 64-byte halves where two rows would start at one bank. Each lane copies the values' pieces that it reads.
    constexpr int CH = 4 * NU;
    auto key_at = [&](int row, int chunk) { return row * CH + (NU % 2 ? chunk : chunk ^ (row & 1) << 2); };
    uint4 *kring = ring - lane;
    auto fetch = [&](int ahead) {
        if (ahead < st1) {
            int s, e;
            step_slots(ahead, s, e);
            uint4 *dst = ring + put * KV * 32, *kdst = kring + put * KV * 32;
            put = put + 1 == FR_DEPTH ? 0 : put + 1;
            // past the end: the last row again, its score masked; past D: zeros
#pragma unroll
            for (int i = 0; i < 2 * NU; i++) {
                const int at = 32 * i + lane, row = at / CH, chunk = at % CH;
                const bool in = 8 * chunk < c.D;
                cp_async16_zfill(kdst + key_at(row, chunk), in ? kb + (size_t)min(s + row, e - 1) * c.D + 8 * chunk : kb, in);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint16_t *row = vb + (size_t)min(s + 2 * cc + (i & 1) + 8 * (i >> 1), e - 1) * c.D + 8 * g;
#pragma unroll
                for (int w = 0; w < NW; w++) {
                    const bool in = 64 * w + 8 * g < c.D;
                    cp_async16_zfill(dst + (2 * NU + 4 * w + i) * 32, in ? row + 64 * w : vb, in);
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < FR_DEPTH - 1; i++) fetch(st0 + i);

    // query fragments: column g (of each column tile), features in the keys' order
    uint4 qb[NT][NU];
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int r = ROWS == 4 ? g & 3 : g + 8 * i;
        const uint16_t *q = c.q + token_of(r) * c.q_stride + (int64_t)qhead_of(r) * c.D + 8 * cc;
#pragma unroll
        for (int u = 0; u < NU; u++)
            qb[i][u] = r < nrows && 32 * u + 8 * cc < c.D ? ldg_nc_v4(q + 32 * u) : make_uint4(0, 0, 0, 0);
    }
    // this lane's columns 2 cc and 2 cc + 1 of a column tile: rows, positions, statistics
    auto row_of = [&](int i, int x) { return ROWS == 4 ? (2 * cc + x) & 3 : 8 * i + 2 * cc + x; };
    int p[NT][2];
    float m[NT][2], l[NT][2], o[NT][NW * 4][4];
#pragma unroll
    for (int i = 0; i < NT; i++) {
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int r = row_of(i, x), at = __shfl_sync(0xffffffffu, rp, r);
            p[i][x] = r < nrows ? at : pmax;
            m[i][x] = -INFINITY;
            l[i][x] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < NW * 4; j++) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
    }
    const float s2 = c.scale * LOG2E;

#pragma unroll 1
    for (int st = st0; st < st1; st++) {
        __syncwarp();                                // the stage has been read
        fetch(st + FR_DEPTH - 1);
        cp_async_wait<FR_DEPTH - 1>();
        __syncwarp();
        const uint4 *src = ring + get * KV * 32, *ks = kring + get * KV * 32;
        get = get + 1 == FR_DEPTH ? 0 : get + 1;
        // scores of keys g and g + 8 (rows) in this lane's columns, as two chains
        float z[NT][4], z1[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) z[i][x] = z1[i][x] = 0.f;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            const uint4 k0 = ks[key_at(g, 4 * u + cc)], k1 = ks[key_at(g + 8, 4 * u + cc)];
            const uint32_t a0[4] = {k0.x, k1.x, k0.y, k1.y}, a1[4] = {k0.z, k1.z, k0.w, k1.w};
#pragma unroll
            for (int i = 0; i < NT; i++) {
                mma_bf16_16816(z[i], a0, qb[i][u].x, qb[i][u].y);
                mma_bf16_16816(z1[i], a1, qb[i][u].z, qb[i][u].w);
            }
        }
        int s, e;
        step_slots(st, s, e);
        const bool edge = s + 16 > e || multi;
        uint32_t ph[NT][2], pl[NT][2];               // weights as B fragments
#pragma unroll
        for (int i = 0; i < NT; i++) {
#pragma unroll
            for (int x = 0; x < 4; x++) z[i][x] += z1[i][x];
            if (edge)
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int key = s + g + 8 * (x >> 1), pr = p[i][x & 1];
                    bool see = key < e;
                    if (multi) {
                        const int kp = slot_pos(c, key);
                        see = see && kp <= pr && (kp >= window_lo(c, pr) || kp < c.sinks);
                    }
                    if (!see) z[i][x] = -INFINITY;
                }
            float mu[2];
            bool grow = false;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                float mx = fmaxf(z[i][x], z[i][2 + x]);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                mu[x] = fmaxf(m[i][x], mx);
                grow = grow || mu[x] > m[i][x];
            }
            if (__any_sync(0xffffffffu, grow))
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float a = mu[x] == -INFINITY ? 1.f : ex2((m[i][x] - mu[x]) * s2);
                    m[i][x] = mu[x];
                    l[i][x] *= a;
#pragma unroll
                    for (int j = 0; j < NW * 4; j++) {
                        o[i][j][x] *= a;
                        o[i][j][2 + x] *= a;
                    }
                }
            float w[4];
#pragma unroll
            for (int x = 0; x < 4; x++) w[x] = ex2((z[i][x] - (mu[x & 1] == -INFINITY ? 0.f : mu[x & 1])) * s2);
#pragma unroll
            for (int k = 0; k < 2; k++) {            // key g, key g + 8
                const uint32_t hi = cvt_bf2(w[2 * k], w[2 * k + 1]);
                if constexpr (LOW) {
                    const uint32_t lo = cvt_bf2(w[2 * k] - lo_bf(hi), w[2 * k + 1] - hi_bf(hi));
                    l[i][0] += w[2 * k];
                    l[i][1] += w[2 * k + 1];
                    ph[i][k] = transpose8(ROWS == 4 && cc >= 2 ? lo : hi);
                    if (ROWS == 8) pl[i][k] = transpose8(lo);
                } else {
                    l[i][0] += lo_bf(hi);
                    l[i][1] += hi_bf(hi);
                    ph[i][k] = transpose8(hi);
                }
            }
        }
#pragma unroll
        for (int w = 0; w < NW; w++) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = src[(2 * NU + 4 * w + i) * 32];
            const uint32_t *y0 = &v[0].x, *y1 = &v[1].x, *y2 = &v[2].x, *y3 = &v[3].x;
#pragma unroll
            for (int j = 0; j < 4; j++) {            // features 2 j (rows g) and 2 j + 1 (rows g + 8)
                const uint32_t a[4] = {__byte_perm(y0[j], y1[j], 0x5410), __byte_perm(y0[j], y1[j], 0x7632),
                                       __byte_perm(y2[j], y3[j], 0x5410), __byte_perm(y2[j], y3[j], 0x7632)};
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    mma_bf16_16816(o[i][4 * w + j], a, ph[i][0], ph[i][1]);
                    if (ROWS == 8) mma_bf16_16816(o[i][4 * w + j], a, pl[i][0], pl[i][1]);
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();                                 // the rings become the warps' results

#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
            // the column's sum over its 8 lanes, then this warp's result to shared memory
            float sum = l[i][x];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            const int r = row_of(i, x);
            if (g == 0 && (ROWS > 4 || cc < 2)) {
                sm[warp * ROWS + r] = m[i][x];
                sl[warp * ROWS + r] = sum;
            }
            float *dst = so + (size_t)(warp * ROWS + r) * DP + 8 * g;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    f[2 * j] = o[i][4 * w + j][x];
                    f[2 * j + 1] = o[i][4 * w + j][2 + x];
                }
                if (ROWS == 4)                       // the low terms' columns
#pragma unroll
                    for (int j = 0; j < 8; j++) f[j] += __shfl_xor_sync(0xffffffffu, f[j], 2);
                if (ROWS > 4 || cc < 2) {
                    *reinterpret_cast<float4 *>(dst + 64 * w) = make_float4(f[0], f[1], f[2], f[3]);
                    *reinterpret_cast<float4 *>(dst + 64 * w + 4) = make_float4(f[4], f[5], f[6], f[7]);
                }
            }
        }
    __syncthreads();
    // the CTA's warps into warp 0's rows
    for (int i = tid; i < nrows * (DP / 4); i += W * 32) {
        const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, sm[w * ROWS + r]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float mw = sm[w * ROWS + r], a = mw == -INFINITY ? 0.f : ex2((mw - M) * s2);
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
        // (a sum that is NaN stays so, whatever its weight)
        for (int w = 0; w < W; w++) {
            const float mw = sm[w * ROWS + tid];
            L = fmaf(sl[w * ROWS + tid], mw == -INFINITY ? 0.f : ex2((mw - M) * s2), L);
        }
        sm[tid] = M;
        sl[tid] = L;
    }
    const int ncl = t.cluster ? ncta : 1;            // CTAs whose results meet here
    if (ncl > 1) cluster_sync_all();
    else __syncthreads();
    pdl_wait();                                      // the prefix half's results
    // weights of the sources (cluster ranks in order, then the prefix's splits): a warp per row
    const int64_t prow = (int64_t)c.n * c.hq;
    const int nsrc = ncl + c.parts;
    for (int r = warp; r < nrows; r += W) {
        const int64_t row = (int64_t)token_of(r) * c.hq + qhead_of(r);
        float mv[FR_SRC / 32], lv[FR_SRC / 32], M = -INFINITY, L = 0.f;
#pragma unroll
        for (int u = 0; u < FR_SRC / 32; u++) {
            const int k = 32 * u + lane;
            mv[u] = -INFINITY;
            lv[u] = 0.f;
            if (k < ncl) {
                mv[u] = ncl > 1 ? ld_cluster(sm + r, k) : sm[r];
                lv[u] = ncl > 1 ? ld_cluster(sl + r, k) : sl[r];
            } else if (k < nsrc) {
                const float2 ml = c.part_ml[(k - ncl) * prow + row];
                mv[u] = ml.x;
                lv[u] = ml.y;
            }
            M = fmaxf(M, mv[u]);
        }
        M = warp_max(M);
#pragma unroll
        for (int u = 0; u < FR_SRC / 32; u++) {
            const float a = mv[u] == -INFINITY ? 0.f : ex2((mv[u] - M) * s2);
            L = fmaf(a, lv[u], L);
            if (32 * u + lane < nsrc) sw[(32 * u + lane) * ROWS + r] = a;
        }
        L = warp_sum(L);
        if (lane == 0) {
            srow[r] = t.part_o ? 1.f : L == 0.f ? 0.f : 1.0f / L;   // a row that sees nothing is zero
            if (t.part_o && rank % ncl == 0) t.part_ml[blockIdx.x / ncl * t.prow + row] = make_float2(M, L);
        }
    }
    __syncthreads();
    // rows x features over the CTAs that met
    const int me = t.cluster ? rank : 0;
    for (int i = me * W * 32 + tid; i < nrows * (c.D / 4); i += ncl * W * 32) {
        const int r = i / (c.D / 4), d = 4 * (i % (c.D / 4)), token = token_of(r), qh = qhead_of(r);
        const int64_t row = (int64_t)token * c.hq + qh;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](const float4 &v, int src) {
            const float a = sw[src * ROWS + r];
            acc.x = fmaf(a, v.x, acc.x);
            acc.y = fmaf(a, v.y, acc.y);
            acc.z = fmaf(a, v.z, acc.z);
            acc.w = fmaf(a, v.w, acc.w);
        };
        const float *mine = so + (size_t)r * DP + d;
        if (ncl == 1) {
            add(*reinterpret_cast<const float4 *>(mine), 0);
        } else {
            for (int k = 0; k < ncl; k += 4) {       // four loads in flight
                float4 v[4];
#pragma unroll
                for (int u = 0; u < 4; u++) v[u] = ld_cluster4(mine, min(k + u, ncl - 1));
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (k + u < ncl) add(v[u], k + u);
            }
        }
        constexpr int PF = 10;                       // splits' loads in flight
        const float *po = c.part_o + row * c.D + d;
        for (int k = 0; k < c.parts; k += PF) {
            float4 v[PF];
#pragma unroll
            for (int u = 0; u < PF; u++) {
                // a split that saw nothing wrote no row
                const bool live = k + u < c.parts && sw[(ncl + k + u) * ROWS + r] != 0.f;
                v[u] = live ? *reinterpret_cast<const float4 *>(po + (k + u) * prow * c.D) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < PF; u++)
                if (k + u < c.parts) add(v[u], ncl + k + u);
        }
        if (t.part_o) {
            *reinterpret_cast<float4 *>(t.part_o + (blockIdx.x / ncl * t.prow + row) * c.D + d) = acc;
        } else {
            const float inv = srow[r];
            *reinterpret_cast<uint2 *>(c.out + token * c.out_stride + (int64_t)qh * c.D + d) =
                make_uint2(cvt_bf2(acc.x * inv, acc.y * inv), cvt_bf2(acc.z * inv, acc.w * inv));
        }
    }
    if (ncl > 1) cluster_sync_all();                 // no CTA leaves while its shared memory is read
}

template <int NU, int ROWS, int W>
static int launch_few(const AttnCall &c, const FewCall &t, int splits, int tiles, bool pdl, cudaStream_t st) {
    auto kern = attend_few_kernel<NU, ROWS, W>;
    const size_t smem = ((size_t)W * (fr_warp_floats(NU, ROWS) + 2 * ROWS) + (FR_SRC + 1) * ROWS) * 4;
    if (!smem_allowed((const void *)kern, smem)) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, c.hkv * tiles, t.tails ? c.n : 1);
    cfg.blockDim = dim3(W * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (t.cluster) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = splits;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        na++;
    }
    if (pdl) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        na++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    MLXD_CHECK(cudaLaunchKernelEx(&cfg, kern, c, t));
    return 0;
}

template <int NU, int W>
static int launch_few_rows(const AttnCall &c, const FewCall &t, int R, int splits, int tiles, bool pdl, cudaStream_t st) {
    return R == 4   ? launch_few<NU, 4, W>(c, t, splits, tiles, pdl, st)
           : R == 8 ? launch_few<NU, 8, W>(c, t, splits, tiles, pdl, st)
                    : launch_few<NU, 16, W>(c, t, splits, tiles, pdl, st);
}
template <int W>
static int launch_few_w(const AttnCall &c, const FewCall &t, int R, int splits, int tiles, bool pdl, cudaStream_t st) {
    if constexpr (W == 4) {                          // (8 such rings exceed an SM's shared memory)
        if (c.D > 192) return launch_few_rows<8, 4>(c, t, R, splits, tiles, pdl, st);
        if (c.D > 128) return launch_few_rows<6, 4>(c, t, R, splits, tiles, pdl, st);
    }
    switch ((c.D + 31) / 32) {
    case 1: return launch_few_rows<1, W>(c, t, R, splits, tiles, pdl, st);
    case 2: return launch_few_rows<2, W>(c, t, R, splits, tiles, pdl, st);
    case 3: return launch_few_rows<3, W>(c, t, R, splits, tiles, pdl, st);
    case 4: return launch_few_rows<4, W>(c, t, R, splits, tiles, pdl, st);
    }
    set_error("attention: head dim %d", c.D);
    return -1;
}

static int launch_join(const AttnCall &c, cudaStream_t st);

// What a few-rows launch is for: the whole result of a cache call; a prefix's
// partial results for a group (into c.part_*); tails, which join them.
enum FewKind { FEW_CACHE, FEW_PREFIX, FEW_TAILS };

// keys: the most that an item reads
static int attend_few(AttnCall &c, FewKind kind, int keys, void *ws, cudaStream_t st) {
    const int64_t rows = kind == FEW_TAILS ? c.rep : (int64_t)c.n * c.rep, qrows = (int64_t)c.n * c.hq;
    const int R = rows > 8 ? 16 : rows > 4 ? 8 : 4;
    const int64_t tiles = (rows + R - 1) / R, items = c.hkv * tiles * (kind == FEW_TAILS ? c.n : 1);
    if (c.hkv * tiles > 65535 || c.n > 65535) {
        set_error("attention: too many rows for one launch");
        return -1;
    }
    FewCall t = {};
    t.tails = kind == FEW_TAILS;
    // CTAs per item: as many as fill the SMs (items enough: three CTAs of 4 warps to an SM; 24 sequences of up to
    // 4096 own tokens 91 us, against 145 with one) while each of their warps has two steps of 16 keys
    const int W = c.D > 128 || items >= num_sms() ? 4 : 8;
    int64_t s = (W == 4 && c.D <= 128 ? 3 : 1) * num_sms() / items;
    if (s > (keys + W * 32 - 1) / (W * 32)) s = (keys + W * 32 - 1) / (W * 32);
    if (s > FR_PARTS) s = FR_PARTS;
    if (s > AT_WS_ROWS / qrows) s = AT_WS_ROWS / qrows;
    if (s < 1) s = 1;
    // more than two clusters' worth: partial results and a second kernel; up to that one cluster, of a power of two
    // (8 kv heads of 32: 4095 positions on 64 CTAs 11.7 us, 8191 on 144 14.9)
    const bool partial = kind == FEW_PREFIX || (kind == FEW_CACHE && s > 2 * FR_MAXCL);
    if (partial) {
        t.prow = qrows;
        t.part_o = (float *)ws;
        t.part_ml = at_ws_ml(ws, c.D);
    } else {
        int cl = 1;
        while (cl < FR_MAXCL && cl * 2 <= s) cl *= 2;
        s = cl;
        t.cluster = cl > 1;
    }
    const bool pdl = kind == FEW_TAILS && c.parts > 0;
    if (W == 4 ? launch_few_w<4>(c, t, R, (int)s, (int)tiles, pdl, st) : launch_few_w<8>(c, t, R, (int)s, (int)tiles, pdl, st))
        return -1;
    if (!partial) return 0;
    c.part_o = t.part_o;
    c.part_ml = t.part_ml;
    c.parts = (int)s;
    return kind == FEW_CACHE ? launch_join(c, st) : 0;
}

// ---- many query rows per kv head: tensor-core tiles
//
// A CTA takes up to 256 query rows of one kv head (the head groups of
// consecutive tokens, or of a batch's sequences: rows r = token * rep + head
// in group, so that a key tile is read once for the whole group) and walks
// the visible slots 128 at a time, in slot order: a ring needs no unwrapping.
//
//   warps 0 and 2, one TMA: key tiles (128 slots x D, 128B swizzle) and value
//   lane each          tiles into their stages (by one lane a key tile waited
//                      behind the values' stage: 512-token chunk 59.8 -> 53.5 us);
//   warp 1             per query tile t (two of 128 rows) and key tile j:
//                      S = Q K^T into TMEM, and once the softmax warps have
//                      put the weights in place of S, O += P V (P from TMEM,
//                      V as stored: its rows are the contraction);
//   warps 4-7, 8-11    query tile 0 / 1, one row per thread: maximum and sum
//                      of S over the key tile, P = e^(S - m) rounded to bf16
//                      over S's own columns. The sum is of the rounded
//                      weights: with a maximum in use below the true one the
//                      largest is not 1, and a row's weights have to sum to
//                      one as they enter the product. O is rescaled only when
//                      a row's maximum grew by more than 2^8 (the statistics
//                      are relative to the maximum in use, so any will do).
//
// While one query tile is in its softmax the tensor cores work on the other.
// Per key tile and 256 rows the MMAs take 2048 clocks and the exponentials as
// many; the chain S -> maximum -> weights -> P V -> S of a query tile leaves some
// 3700 (tensor pipe and exponentials 57% busy). A 4096-token chunk at 4096 of
// 32/8 heads takes 374 us, 1102 TFLOP/s, 65% of the cuBLAS burst rate, in runs of
// a few ms, and 430 us (960 TFLOP/s) in seconds of them, at the power limit (985 W,
// 1.7 GHz); with the softmax left out the same MMAs took 328 us. The softmax warps
// spill 20 to 70 bytes a thread. The first weights are taken by the old maximum
// while the new one is found, and again when it grew (398 -> 384 us). Tried without gain: exponentials of every
// 3rd or 4th pair as a cubic on the FMA pipe, a row shared by two threads (500
// us: four softmax warps to a scheduler wait for each other's maxima), the MMAs
// of whichever tile is ready (704 us: both fall into phase), weights stored 32
// keys at a time (402 us), three key or value stages.
// Keys no row of the CTA sees may hold anything: their scores are masked and
// their value rows zeroed in shared memory. Every wait is bounded; a launch
// that gave up says so in its cache's (or group's) host word, which the next
// call over it reports.
constexpr int AT_THREADS = 384, AT_KT = 128, AT_ROWS = 256;

template <int DB, bool BK>
struct AtLayout {
    static constexpr int KS = DB == 1 ? 3 : 2, VS = KS;   // stages (a third of 128 features gains nothing)
    static constexpr int BLOCK = AT_KT * 128;          // 128 rows x 64 features
    static constexpr int TILE = DB * BLOCK;
    static constexpr size_t Q = 0, K = (BK ? 1 : 2) * TILE, V = K + KS * TILE, BARS = V + VS * TILE;
    static constexpr size_t TOTAL = 1024 + BARS + 512;
};

struct TileCall {
    int z0;                    // the layer's first kv head in the tensor maps
    int splits;                // key splits (grid z)
    float *part_o;             // partial results, or null: the whole result to out
    float2 *part_ml;
    int64_t prow;              // rows per split of the partial results
    int *fail;
};

// bits x of a 32-slot word at s0 with lo <= s0 + x < hi
MLXD_DEV uint32_t span_bits(int s0, int lo, int hi) {
    const int l = min(max(lo - s0, 0), 32), h = min(max(hi - s0, 0), 32);
    const uint32_t up = h == 32 ? 0xffffffffu : (1u << h) - 1u;
    return l >= h ? 0u : up & (0xffffffffu << l);
}
// BK: a CTA takes 128 rows, its two softmax halves alternating key tiles
template <int DB, bool BK>
__global__ void __launch_bounds__(AT_THREADS, 1)
    attend_tile_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                       const __grid_constant__ AttnCall c, const __grid_constant__ TileCall t) {
    using L = AtLayout<DB, BK>;
    constexpr int KS = L::KS, VS = L::VS;
    extern __shared__ __align__(1024) unsigned char at_raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>(((uintptr_t)at_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *kfull = reinterpret_cast<uint64_t *>(sm + L::BARS);
    uint64_t *kempty = kfull + KS, *vfull = kempty + KS, *vempty = vfull + VS;
    uint64_t *sfull = vempty + VS, *pfull = sfull + 2, *qfull = pfull + 4, *odone = qfull + 1, *xdone = odone + 1;   // pfull[2 t + half]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(xdone + 1);
    __shared__ int s_min[8], s_max[8], s_fail;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // Several waves: the longest rows of all heads first (a head after another: 4096-token chunk 384 us, against
    // 379). One wave: a head's tiles side by side, which share its keys' way to the SMs.
    const int rows = c.n * c.rep, head = BK ? blockIdx.y : blockIdx.x;
    const int r0 = BK ? (gridDim.x - 1 - blockIdx.x) * 128 : (gridDim.y - 1 - blockIdx.y) * AT_ROWS;
    const int nq = BK || rows - r0 > 128 ? 2 : 1;
    if (tid == 0) {
        for (int i = 0; i < 2 * (KS + VS); i++) mbar_init(&kfull[i], 1);
        for (int i = 0; i < 2; i++) mbar_init(&sfull[i], 1);
        for (int i = 0; i < 4; i++) mbar_init(&pfull[i], 4);
        mbar_init(qfull, 8);
        mbar_init(odone, 1);
        mbar_init(xdone, 4);
        s_fail = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp >= 4) {                                 // positions of the CTA's 256 rows
        const int i = tid - 128, r = r0 + (BK ? i & 127 : i), p = r < rows ? query_pos(c, r / c.rep) : -1;
        const int lo = __reduce_min_sync(0xffffffffu, p < 0 ? INT32_MAX : p), hi = __reduce_max_sync(0xffffffffu, p);
        if (lane == 0) {
            s_min[warp - 4] = lo;
            s_max[warp - 4] = hi;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();   // every CTA is on an SM: the tails may start on free ones
    int pmin = s_min[0], pmax = s_max[0];
#pragma unroll
    for (int i = 1; i < 8; i++) {
        pmin = min(pmin, s_min[i]);
        pmax = max(pmax, s_max[i]);
    }

    // the visible slots as tiles: sinks, a ring's wrapped end, the rest
    int a1 = 0, c0 = 0, c1 = 0, b0 = 0, b1 = 0;      // tile ranges [0, a1), [c0, c1), [b0, b1)
    Span all = {0, 0, 0, 0, 0};                      // the slots any row sees
    if (pmax >= 0) {
        all = span_of(c, window_lo(c, pmin), pmax + 1);
        a1 = (all.a1 + AT_KT - 1) / AT_KT;
        if (all.c1 > all.c0) {
            c0 = max(all.c0 / AT_KT, a1);
            c1 = max((all.c1 + AT_KT - 1) / AT_KT, c0);
        }
        if (all.b1 > all.b0) {
            b0 = max(all.b0 / AT_KT, max(a1, c1));
            b1 = max((all.b1 + AT_KT - 1) / AT_KT, b0);
        }
    }
    const int nt = a1 + (c1 - c0) + (b1 - b0);
    const int j0 = (int)((int64_t)nt * blockIdx.z / t.splits), j1 = (int)((int64_t)nt * (blockIdx.z + 1) / t.splits);
    // key tile n of query tile i, counted from j0
    auto key_tile = [&](int i, int n) { return BK ? 2 * n + i : n; };
    auto tile_slot = [&](int j) {
        const int k = j < a1 ? j : j < a1 + c1 - c0 ? c0 + j - a1 : b0 + j - a1 - (c1 - c0);
        return k * AT_KT;
    };

    // registers to the softmax warps: 128 x (72 + 2 x 208) of the block's 384 x 168
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if ((warp == 0 || warp == 2) && lane == 0) {   // the keys' loads, the values' loads
            auto loads = [&](const CUtensorMap &tm, uint64_t *full, uint64_t *empty, size_t base, auto stages) {
                constexpr int NS = decltype(stages)::value;
                const uint64_t map = reinterpret_cast<uint64_t>(&tm);
                int n = 0;                           // loads issued
                for (int j = j0; j < j1; j++) {
                    const int st = n % NS, u = n / NS;
                    if (u > 0 && !mbar_wait(&empty[st], (u - 1) & 1)) {
                        s_fail = 1;
                        break;
                    }
                    mbar_expect_tx(&full[st], L::TILE);
                    n++;
#pragma unroll
                    for (int b = 0; b < DB; b++)
                        asm volatile(
                            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                            ::"r"(smem_u32(sm + base + st * L::TILE + b * L::BLOCK)), "l"(map), "r"(b * 64),
                            "r"(tile_slot(j)), "r"(t.z0 + head), "r"(smem_u32(&full[st]))
                            : "memory");
                }
                // after a failure: no copy may land once the CTA is gone
                for (int i = 0; i < NS; i++)
                    if (n > i) mbar_wait(&full[(n - 1 - i) % NS], ((n - 1 - i) / NS) & 1);
            };
            if (warp == 0) loads(tmk, kfull, kempty, L::K, std::integral_constant<int, KS>());
            else loads(tmv, vfull, vempty, L::V, std::integral_constant<int, VS>());
        } else if (warp == 1 && j1 > j0) {
            constexpr uint32_t iqk = umma_idesc_bf16(128, AT_KT, false), ipv = umma_idesc_bf16(128, DB * 64, true);
            const uint64_t qd = umma_desc_sw128(smem_u32(sm + L::Q)), kd = umma_desc_sw128(smem_u32(sm + L::K));
            const uint64_t vd = umma_desc_sw128_mn(smem_u32(sm + L::V), L::BLOCK);
            auto qk = [&](int i, int n) {            // S_i = Q_i K_n^T
                const uint64_t qt = qd + (BK ? 0 : i * (L::TILE >> 4)), kt = kd + (n % KS) * (L::TILE >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < DB * 4; k++) {
                        const uint64_t off = ((k >> 2) * L::BLOCK + (k & 3) * 32) >> 4;
                        mma_ss(tmem + i * 128, qt + off, kt + off, iqk, k != 0);
                    }
                    tc_commit(&sfull[i]);
                }
            };
            auto pv = [&](int i, int n, int half, bool add) {  // O_i += P_i V_n over 64 keys
                const uint64_t vt = vd + (n % VS) * (L::TILE >> 4) + half * (4 * 2048 >> 4);
                const uint32_t pt = tmem + i * 128 + half * 32;
                if (elect_one())
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        mma_ts(tmem + 256 + i * 128, pt + k * 8, vt + (k * 2048 >> 4), ipv, add || half + k != 0);
            };
            auto release = [&](uint64_t *bar) {
                if (elect_one()) tc_commit(bar);
            };
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                const bool got = __all_sync(0xffffffffu, mbar_wait(bar, parity));
                tc_fence_after();
                return got;
            };
            // the query tiles strictly in turn, which keeps one in its softmax while the other multiplies; a
            // key tile is waited for by its first user and released by its last
            const int nn = j1 - j0;
            auto first = [&](int i) { return BK || i == 0; };
            auto last = [&](int i) { return BK || i == nq - 1; };
            bool ok = wait(qfull, 0);
            auto scores = [&](int i, int n) {
                const int k = key_tile(i, n);
                if (!ok || k >= nn) return;
                if (first(i) && !(ok = wait(&kfull[k % KS], (k / KS) & 1))) return;
                qk(i, k);
                if (last(i)) release(&kempty[k % KS]);
            };
            for (int i = 0; i < nq; i++) scores(i, 0);
            for (int n = 0; key_tile(0, n) < nn && ok; n++)
                for (int i = 0; i < nq; i++) {
                    const int k = key_tile(i, n);
                    if (k >= nn) break;
                    if (first(i)) ok = ok && wait(&vfull[k % VS], (k / VS) & 1);
                    for (int h = 0; h < 2 && ok; h++)
                        if ((ok = wait(&pfull[2 * i + h], n & 1))) pv(i, k, h, n > 0);
                    if (ok && last(i)) release(&vempty[k % VS]);
                    scores(i, n + 1);
                }
            release(odone);
            if (!wait(odone, 0) || !ok) s_fail = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // the query tiles (zero past the rows and D), K-major in the 128B swizzle: a warp's rows, whose addresses
        // its lanes hold, in 16-byte chunks with all loads in flight
        {
            constexpr int RW = (BK ? 128 : AT_ROWS) / 8, PER = RW * DB / 4;
            const int w0 = (warp - 4) * RW, mine = r0 + w0 + lane, tok = mine / c.rep;
            const uint16_t *src = c.q + tok * c.q_stride + (int64_t)(head * c.rep + mine - tok * c.rep) * c.D;
            uint4 v[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int r = i * (4 / DB) + lane / (DB * 8), ch = lane % (DB * 8);
                const uint16_t *at = reinterpret_cast<const uint16_t *>(__shfl_sync(0xffffffffu, (unsigned long long)src, r));
                v[i] = r0 + w0 + r < rows && ch * 8 < c.D ? ldg_nc_v4(at + ch * 8) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int r = w0 + i * (4 / DB) + lane / (DB * 8), ch = lane % (DB * 8);
                *reinterpret_cast<uint4 *>(sm + L::Q + (r >> 7) * L::TILE + (ch >> 3) * L::BLOCK + (r & 127) * 128 +
                                           (((ch & 7) ^ (r & 7)) << 4)) = v[i];
            }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);

        if ((warp - 4) / 4 < nq) {
        const int wg = (warp - 4) >> 2, trow = (warp & 3) * 32 + lane, row = r0 + (BK ? 0 : wg * 128) + trow;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + wg * 128, to = tmem + lanes + 256 + wg * 128;
        const float s2 = c.scale * LOG2E, slack = 8.0f / s2;
        const int token = row / c.rep;
        const int p = row < rows ? query_pos(c, token) : -1;
        // what this row sees; rows that are not asked for see all (and are dropped)
        Span sp = {0, 0, 0, 0, INT32_MAX};
        if (p >= 0) sp = span_of(c, window_lo(c, p), p + 1);
        float m = -INFINITY;
        uint64_t l[2] = {pair2(0.f, 0.f), pair2(0.f, 0.f)};   // the row sum, in four
        bool ok = true;
        for (int n = 0; key_tile(wg, n) < j1 - j0; n++) {
            const int k = key_tile(wg, n), s0 = tile_slot(j0 + k);
            uint32_t see[4] = {~0u, ~0u, ~0u, ~0u};
            bool whole = s0 >= sp.b0 && s0 + AT_KT <= sp.b1;
            if (!whole)
#pragma unroll
                for (int w = 0; w < 4; w++)
                    see[w] = span_bits(s0 + 32 * w, 0, sp.a1) | span_bits(s0 + 32 * w, sp.c0, sp.c1) |
                             span_bits(s0 + 32 * w, sp.b0, sp.b1);
            whole = __all_sync(0xffffffffu, (see[0] & see[1] & see[2] & see[3]) == ~0u);
            if (!__all_sync(0xffffffffu, mbar_wait(&sfull[wg], n & 1))) {
                s_fail = 1;
                ok = false;
                break;
            }
            tc_fence_after();
            uint32_t v[4][32];
            auto mask = [&](int w) {
#pragma unroll
                for (int x = 0; x < 32; x++) v[w][x] = see[w] >> x & 1 ? v[w][x] : 0xff800000u;
            };
            // weights of 32 keys relative to the maximum in use, and their sums
            uint32_t pk[32];
            float add[4];
            auto weigh = [&](int w) {
                const float mu = m == -INFINITY ? 0.f : m * s2;
                const uint64_t ss = pair2(s2, s2), mm = pair2(-mu, -mu);
                if (!(w & 1)) add[0] = add[1] = add[2] = add[3] = 0.f;
#pragma unroll
                for (int x = 16 * (w & 1); x < 16 * (w & 1) + 16; x++) {
                    const int y = 2 * (x % 16);
                    float e0, e1;
                    unpair2(fma2(pair2(__uint_as_float(v[w][y]), __uint_as_float(v[w][y + 1])), ss, mm), e0, e1);
                    e0 = ex2(e0);
                    e1 = ex2(e1);
                    pk[x] = cvt_bf2(e0, e1);
                    add_bf2(add[2 * (x & 1)], add[2 * (x & 1) + 1], pk[x]);
                }
            };
#pragma unroll
            for (int w = 0; w < 4; w++) tmem_ld32(v[w], ts + 32 * w);
            tmem_wait_ld();
            if (!whole)
#pragma unroll
                for (int w = 0; w < 4; w++) mask(w);
            weigh(0);                                // by the old maximum, which mostly stays
            float mw[4];
#pragma unroll
            for (int w = 0; w < 4; w++) {
                mw[w] = __uint_as_float(v[w][0]);
#pragma unroll
                for (int x = 1; x < 32; x++) mw[w] = fmaxf(mw[w], __uint_as_float(v[w][x]));
            }
            const float mx = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
            // a new maximum only when the old one is too far below
            const bool grow = mx > m + slack || (m == -INFINITY && mx > -INFINITY);
            if (__any_sync(0xffffffffu, grow)) {
                const float a = grow ? ex2((m - mx) * s2) : 1.0f;
                if (grow) m = mx;
                l[0] = mul2(l[0], pair2(a, a));
                l[1] = mul2(l[1], pair2(a, a));
                if (n > 0)
#pragma unroll
                    for (int w = 0; w < DB * 4; w++) {
                        uint32_t o[16];
                        tmem_ld16(o, to + 16 * w);
                        tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * a);
                        tmem_st16(to + 16 * w, o);
                    }
                weigh(0);
            }
            // value rows of slots that no row sees: whatever they hold must not meet a zero weight
            if ((BK || wg == 0) && !(s0 >= all.b0 && s0 + AT_KT <= all.b1)) {
                if (!__all_sync(0xffffffffu, mbar_wait(&vfull[k % VS], (k / VS) & 1))) {
                    s_fail = 1;
                    ok = false;
                    break;
                }
                const int s = s0 + trow;
                if (!(s < all.a1 || (s >= all.c0 && s < all.c1) || (s >= all.b0 && s < all.b1)))
#pragma unroll
                    for (int b = 0; b < DB; b++)
#pragma unroll
                        for (int q = 0; q < 8; q++)
                            *reinterpret_cast<uint4 *>(sm + L::V + (k % VS) * L::TILE + b * L::BLOCK + trow * 128 + q * 16) =
                                make_uint4(0, 0, 0, 0);
                fence_proxy_async();
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (h == 1) weigh(2);
                weigh(2 * h + 1);
                l[0] = add2(l[0], pair2(add[0], add[1]));
                l[1] = add2(l[1], pair2(add[2], add[3]));
                tmem_st32(ts + 32 * h, pk);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[2 * wg + h]);
            }
        }
        float lsum;
        {
            float t;
            unpair2(add2(l[0], l[1]), lsum, t);
            lsum += t;
        }
        const bool have = key_tile(wg, 0) < j1 - j0;
        if (ok && have && !__all_sync(0xffffffffu, mbar_wait(odone, 0))) {
            s_fail = 1;
            ok = false;
        }
        tc_fence_after();
        // by keys: the second half's statistics and O meet the first's through the key and value stages, which
        // nothing uses any more ([feature][row], then maxima and sums)
        float *xo = reinterpret_cast<float *>(sm + L::K), *xm = xo + DB * 64 * 128, *xl = xm + 128;
        float a0 = 1.f, a1 = 0.f;                    // weights of this half's and the other's O
        const bool two = BK && key_tile(1, 0) < j1 - j0;
        if (two && wg == 1 && ok) {
            xm[trow] = m;
            xl[trow] = lsum;
#pragma unroll
            for (int w = 0; w < DB * 2; w++) {
                uint32_t v[32];
                tmem_ld32(v, to + 32 * w);
                tmem_wait_ld();
#pragma unroll
                for (int x = 0; x < 32; x++) xo[(32 * w + x) * 128 + trow] = __uint_as_float(v[x]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(xdone);
        }
        if (BK && wg == 1) ok = false;        // the first half writes
        if (two && wg == 0 && ok) {
            if (!__all_sync(0xffffffffu, mbar_wait(xdone, 0))) {
                s_fail = 1;
                ok = false;
            } else {
                const float m1 = xm[trow], mm = fmaxf(m, m1);
                a0 = m == -INFINITY ? 0.f : ex2((m - mm) * s2);
                a1 = m1 == -INFINITY ? 0.f : ex2((m1 - mm) * s2);
                lsum = a0 * lsum + a1 * xl[trow];
                m = mm;
            }
        }
        if (ok) {
            const int qh = head * c.rep + row - token * c.rep;
            const int64_t prow = (int64_t)token * c.hq + qh;
            const bool live = p >= 0;
            const float inv = t.part_o ? 1.f : lsum == 0.f ? 0.f : 1.0f / lsum;
            if (live && t.part_o) t.part_ml[blockIdx.z * t.prow + prow] = make_float2(have ? m : -INFINITY, have ? lsum : 0.f);
            // 32 columns at a time through shared memory (rows of 36 floats, in the value stages), so that 8
            // lanes write one row's
            float *stage = reinterpret_cast<float *>(sm + L::V + 4096) + (warp - 4) * 32 * 36;
            char *dst = t.part_o ? reinterpret_cast<char *>(t.part_o + (blockIdx.z * t.prow + prow) * c.D)
                                 : reinterpret_cast<char *>(c.out + token * c.out_stride + (int64_t)qh * c.D);
            if (!live) dst = nullptr;
#pragma unroll 1
            for (int w = 0; w < DB * 2 && have; w++) {
                uint32_t v[32];
                tmem_ld32(v, to + 32 * w);
                tmem_wait_ld();
                if (two) {
#pragma unroll
                    for (int x = 0; x < 32; x++)
                        v[x] = __float_as_uint(fmaf(a0, __uint_as_float(v[x]), a1 * xo[(32 * w + x) * 128 + trow]));
                }
#pragma unroll
                for (int x = 0; x < 32; x++) v[x] = __float_as_uint(__uint_as_float(v[x]) * inv);
                __syncwarp();
#pragma unroll
                for (int x = 0; x < 32; x += 4)
                    *reinterpret_cast<uint4 *>(stage + lane * 36 + x) = make_uint4(v[x], v[x + 1], v[x + 2], v[x + 3]);
                __syncwarp();
                const int f = 32 * w + (lane & 7) * 4;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = 4 * i + (lane >> 3);
                    char *at = reinterpret_cast<char *>(__shfl_sync(0xffffffffu, (unsigned long long)dst, r));
                    const float4 o = *reinterpret_cast<const float4 *>(stage + r * 36 + (lane & 7) * 4);
                    if (!at || f >= c.D) continue;
                    if (t.part_o) *reinterpret_cast<float4 *>(at + f * 4) = o;
                    else *reinterpret_cast<uint2 *>(at + f * 2) = make_uint2(cvt_bf2(o.x, o.y), cvt_bf2(o.z, o.w));
                }
            }
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
    if (tid == 0 && s_fail && t.fail) *reinterpret_cast<volatile int *>(t.fail) = 1;
}

// splits of every query row into its output row: one warp per row
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttnCall c) {
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), prow = (int64_t)c.n * c.hq;
    if (row >= prow) return;
    // lane k holds the weights of splits k and k + 32; the features are 4 a lane
    const float s2 = c.scale * LOG2E;
    float w[2], M = -INFINITY, L = 0.f;
    float2 ml[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int k = 32 * u + lane;
        ml[u] = k < c.parts ? c.part_ml[k * prow + row] : make_float2(-INFINITY, 0.f);
        M = fmaxf(M, ml[u].x);
    }
    M = warp_max(M);
#pragma unroll
    for (int u = 0; u < 2; u++) {
        w[u] = ml[u].x == -INFINITY ? 0.f : ex2((ml[u].x - M) * s2);
        L = fmaf(w[u], ml[u].y, L);
    }
    L = warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    constexpr int JOIN = 10;                         // loads in flight
    for (int d = lane * 4; d - lane * 4 < c.D; d += 128) {
        const float *po = c.part_o + row * c.D + d;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < c.parts; k += JOIN) {
            float4 v[JOIN];
            float a[JOIN];
#pragma unroll
            for (int u = 0; u < JOIN; u++) {
                const float lo = __shfl_sync(0xffffffffu, w[0], (k + u) & 31), hi = __shfl_sync(0xffffffffu, w[1], (k + u) & 31);
                a[u] = k + u >= c.parts ? 0.f : k + u < 32 ? lo : hi;
                // a split that saw nothing wrote no row
                v[u] = d < c.D && a[u] != 0.f ? *reinterpret_cast<const float4 *>(po + (k + u) * prow * c.D)
                                              : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < JOIN; u++) {
                acc.x = fmaf(a[u], v[u].x, acc.x);
                acc.y = fmaf(a[u], v[u].y, acc.y);
                acc.z = fmaf(a[u], v[u].z, acc.z);
                acc.w = fmaf(a[u], v[u].w, acc.w);
            }
        }
        if (d < c.D)
            *reinterpret_cast<uint2 *>(c.out + row / c.hq * c.out_stride + row % c.hq * c.D + d) =
                make_uint2(cvt_bf2(acc.x * inv, acc.y * inv), cvt_bf2(acc.z * inv, acc.w * inv));
    }
}

static int launch_join(const AttnCall &c, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((int64_t)c.n * c.hq + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    MLXD_CHECK(cudaLaunchKernelEx(&cfg, attend_join_kernel, c));
    return 0;
}

template <int DB, bool BK>
static int launch_tile(const AttnCall &c, const TileCall &t, const CUtensorMap &mk, const CUtensorMap &mv,
                       cudaStream_t st) {
    auto kern = attend_tile_kernel<DB, BK>;
    if (!smem_allowed((const void *)kern, (AtLayout<DB, BK>::TOTAL))) return -1;
    const int per = BK ? 128 : AT_ROWS, blocks = (c.n * c.rep + per - 1) / per;
    const dim3 grid(BK ? blocks : c.hkv, BK ? c.hkv : blocks, t.splits);
    kern<<<grid, AT_THREADS, (AtLayout<DB, BK>::TOTAL), st>>>(mk, mv, c, t);
    MLXD_CHECK(cudaGetLastError());
    return 0;
}

// The shape of a tile launch. A CTA of 128 rows whose halves alternate key
// tiles takes about half the time of one of 256 rows whose halves share every
// key tile. While the former fit one wave they are taken (a 512-token chunk
// over a 4096 window 60 us, against 69 in 256 rows and two splits, when this
// was chosen; 51 now), beyond it
// the latter, with half the loads per product (a 4096-token chunk 415 us, against
// 514). The step between them is steep: over a 4096 window 576 tokens of 32/8
// heads (144 CTAs of 128 rows) take 50 us, 640 (80 of 256) 84, as 1024 do. Key
// splits fill the SMs when even those are few, no more than the key tiles or the
// workspace's rows.
struct TileShape {
    int by_keys, splits;
};
static TileShape tile_shape(const AttnCall &c, int keys) {
    const int64_t R = (int64_t)c.n * c.rep, rows = (int64_t)c.n * c.hq, sms = num_sms();
    const int64_t pairs = (R + AT_ROWS - 1) / AT_ROWS * c.hkv, singles = (R + 127) / 128 * c.hkv;
    TileShape f;
    f.by_keys = singles <= sms;
    int64_t s = sms / (f.by_keys ? singles : pairs);
    if (s > (keys + AT_KT - 1) / AT_KT) s = (keys + AT_KT - 1) / AT_KT;
    if (s > AT_WS_ROWS / rows) s = AT_WS_ROWS / rows;
    if (s > FR_PARTS) s = FR_PARTS;
    f.splits = s < 1 ? 1 : (int)s;
    return f;
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

// reports once that a launch over this cache or group gave up on a wait
static bool gave_up(int *word, const char *what) {
    volatile int *w = word;
    if (!w || !*w) return false;
    *w = 0;
    set_error("%s: an earlier attention launch over these rows gave up waiting on its pipeline", what);
    return true;
}

// 128 slots x 64 features of [layers * heads][cap][D] bf16 rows, 128B swizzle,
// zero past D and cap
static bool row_map(CUtensorMap *m, const uint16_t *base, int heads, int cap, int D) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)cap, (cuuint64_t)heads};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)cap * D * 2};
    cuuint32_t box[3] = {64, AT_KT, 1}, estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

void kv_attend_prepare(mlxd_kv *kv) {
    // (no tiles without the word that reports their failures)
    kv->gave_up = host_word();
    kv->maps = kv->gave_up && kv->d % 8 == 0 && kv->d <= 128 && row_map(&kv->map_k, kv->k, kv->layers * kv->hkv, kv->cap, kv->d) &&
               row_map(&kv->map_v, kv->v, kv->layers * kv->hkv, kv->cap, kv->d);
}

static int attend_tiles(const AttnCall &c, const mlxd_kv *kv, int layer, TileShape shape, bool partial, void *ws,
                        int *fail, cudaStream_t st) {
    if (!kv->maps) {
        set_error("attention: the cache has no tensor maps (no cuTensorMapEncodeTiled, or no pinned host memory)");
        return -1;
    }
    TileCall t = {};
    t.z0 = layer * kv->hkv;
    t.splits = shape.splits;
    t.prow = (int64_t)c.n * c.hq;
    if (partial) {
        t.part_o = (float *)ws;
        t.part_ml = at_ws_ml(ws, c.D);
    }
    t.fail = fail;
    if (c.D <= 64)
        return shape.by_keys ? launch_tile<1, true>(c, t, kv->map_k, kv->map_v, st)
                             : launch_tile<1, false>(c, t, kv->map_k, kv->map_v, st);
    return shape.by_keys ? launch_tile<2, true>(c, t, kv->map_k, kv->map_v, st)
                         : launch_tile<2, false>(c, t, kv->map_k, kv->map_v, st);
}

static int attend_cache(AttnCall c, const mlxd_kv *kv, int layer, void *ws, cudaStream_t st) {
    const int64_t span = (int64_t)c.window + c.n - 1 + c.sinks, rows = (int64_t)c.n * c.rep;
    const int keys = c.window && span < c.total ? (int)span : c.total;   // the most that one row group sees
    // more than 8 rows per kv head: tiles (16 rows at 8192 positions 18.4 us, against 21.8 with 16 columns of
    // the few-rows kernel; 8 rows 16.9, against 17.5 on tiles)
    if (c.D <= 128 && rows > 8) {
        if (rows > 65535 * AT_ROWS || c.hkv > 65535) {   // the grid's limits
            set_error("kv_attend: too many query rows");
            return -1;
        }
        const TileShape shape = tile_shape(c, keys);
        if (attend_tiles(c, kv, layer, shape, shape.splits > 1, ws, kv->gave_up, st)) return -1;
        if (shape.splits == 1) return 0;
        c.part_o = (const float *)ws;
        c.part_ml = at_ws_ml(ws, c.D);
        c.parts = shape.splits;
        return launch_join(c, st);
    }
    // few rows, or heads wider than 128, for which the tiles have no form (two query tiles' accumulators would fill
    // the TMEM; 4096 tokens at 4096 of 16/2 heads of 256 take 7.96 ms here, 52 TFLOP/s): tokens in launches of at most
    // 65535 items
    int64_t most = (int64_t)(65535 / c.hkv) * 16 / c.rep;
    most = most < 1 ? 1 : most > 65535 ? 65535 : most;
    const int n = c.n;
    for (int i = 0; i < n; i += (int)most) {
        AttnCall b = c;
        b.n = n - i < most ? n - i : (int)most;
        b.q += i * c.q_stride;
        b.out += i * c.out_stride;
        b.pos0 += i;
        if (attend_few(b, FEW_CACHE, keys, ws, st)) return -1;
    }
    return 0;
}

// sequences in batches whose partial rows fit the workspace: the prefix (on
// tiles unless the heads are too wide), then every sequence's tail, which joins the prefix's results
static int attend_group(AttnCall c, const mlxd_kv *kv, int layer, void *ws, int *fail, cudaStream_t st) {
    const int64_t tail = (int64_t)c.hkv * c.tcap * c.D;
    int64_t most = AT_WS_ROWS / c.hq < 65535 ? AT_WS_ROWS / c.hq : 65535;
    if (most < 1) {
        set_error("kv_group_attend: %d query heads", c.hq);
        return -1;
    }
    const int n = c.n;
    for (int64_t i = 0; i < n; i += most) {
        AttnCall b = c;
        b.n = (int)(n - i < most ? n - i : most);
        b.q += i * c.q_stride;
        b.out += i * c.out_stride;
        b.lens += i;
        b.tk += i * tail;
        b.tv += i * tail;
        if (c.prefix > 0 && c.D > 128) {
            if (attend_few(b, FEW_PREFIX, c.prefix, ws, st)) return -1;
        } else if (c.prefix > 0) {
            const TileShape shape = tile_shape(b, c.prefix);
            if (attend_tiles(b, kv, layer, shape, true, ws, fail, st)) return -1;
            b.part_o = (const float *)ws;
            b.part_ml = at_ws_ml(ws, c.D);
            b.parts = shape.splits;
        }
        if (attend_few(b, FEW_TAILS, c.tcap, nullptr, st)) return -1;
    }
    return 0;
}

// the checks that both calls share; fills the call's common half
static int attn_call(AttnCall &c, const char *what, int hkv, int D, const void *q, int64_t q_stride, int n,
                     const mlxd_attn *a, void *out, int64_t out_stride, const void *ws, size_t ws_bytes) {
    if (!a || a->n_heads <= 0 || a->n_heads % hkv || a->window < 0 || a->sinks < 0 || !(a->scale >= 0.f) ||
        a->scale > 1e30f || (a->scale > 0.f && a->scale < 1e-30f)) {
        set_error("%s: bad attention parameters (heads a multiple of %d, window and sinks not negative, scale 0 or 1e-30 .. 1e30)",
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
    if (!on_device(q, "attention: q", 16) || !on_device(out, "attention: out", 16) ||
        !on_device(ws, "attention: workspace", 256))
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
    return head_dim > 0 ? at_ws_bytes(head_dim) : 0;
}

int mlxd_cuda_kv_attend(const mlxd_kv *kv, int layer, const void *q, int64_t q_stride, int n, int pos,
                        const mlxd_attn *a, void *out, int64_t out_stride, void *ws, size_t ws_bytes, void *stream) try {
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
    // of what the queries see, the lowest position that no sink slot keeps
    const int lo = window_lo(c, pos), low = lo <= kv->sinks || c.sinks > kv->sinks ? kv->sinks : lo;
    if (const char *why = kv->missing(layer, low, total, is_capturing((cudaStream_t)stream))) {
        set_error("kv_attend: positions %d to %d of layer %d %s", low, total - 1, layer, why);
        return -1;
    }
    if (!same_device(kv->device, "kv_attend") || gave_up(kv->gave_up, "kv_attend")) return -1;
    const size_t layer_elems = (size_t)kv->hkv * kv->cap * kv->d;
    c.k = kv->k + layer * layer_elems;
    c.v = kv->v + layer * layer_elems;
    c.cap = kv->cap;
    c.ring_sinks = kv->sinks;
    c.pos0 = pos;
    c.total = total;
    return attend_cache(c, kv, layer, ws, (cudaStream_t)stream);
} catch (...) {   // no exception leaves a C entry
    set_error("kv_attend: out of host memory");
    return -1;
}

int mlxd_cuda_kv_group_create(mlxd_kv_group **out, const mlxd_kv *prefix, int prefix_len, int n_seqs,
                              int tail_capacity) try {
    if (!out || !prefix || prefix_len < 0 || prefix_len > prefix->cap || n_seqs <= 0 || tail_capacity <= 0 ||
        (int64_t)prefix_len + tail_capacity > INT32_MAX || prefix->d % 8 || prefix->d > 256) {
        set_error("kv_group_create: bad arguments");
        return -1;
    }
    if (prefix_len > prefix->sinks)
        for (int l = 0; l < prefix->layers; l++)
            if (prefix->held[l].lost > prefix->sinks) {
                set_error("kv_group_create: the prefix of layer %d has been overwritten by later positions", l);
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
    if (!(g->gave_up = host_word())) {
        set_error("kv_group_create: no pinned host memory");
        mlxd_cuda_kv_group_destroy(g);
        return -1;
    }
    *out = g;
    return 0;
} catch (...) {   // no exception leaves a C entry
    set_error("kv_group_create: out of host memory");
    return -1;
}

void mlxd_cuda_kv_group_destroy(mlxd_kv_group *g) {
    if (!g) return;
    cudaDeviceSynchronize();
    dev_free(g->k);
    dev_free(g->v);
    host_word_free(g->gave_up);
    delete g;
}

int32_t *mlxd_cuda_kv_gave_up(const mlxd_kv *kv) { return kv ? kv->gave_up : nullptr; }
int32_t *mlxd_cuda_kv_group_gave_up(const mlxd_kv_group *g) { return g ? g->gave_up : nullptr; }

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
        !on_device(lens_dev, "kv_group_append: lengths", 4) || !same_device(g->device, "kv_group_append"))
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
                              size_t ws_bytes, void *stream) try {
    if (!g || layer < 0 || layer >= g->layers) {
        set_error("kv_group_attend: bad arguments");
        return -1;
    }
    if (const char *why = g->prefix->missing(layer, g->prefix->sinks, g->prefix_len, is_capturing((cudaStream_t)stream))) {
        set_error("kv_group_attend: positions of the prefix of %d in layer %d %s", g->prefix_len, layer, why);
        return -1;
    }
    AttnCall c = {};
    if (attn_call(c, "kv_group_attend", g->hkv, g->d, q, q_stride, g->n, a, out, out_stride, ws, ws_bytes) ||
        !on_device(lens_dev, "kv_group_attend: lengths", 4) || !same_device(g->device, "kv_group_attend") ||
        gave_up(g->gave_up, "kv_group_attend"))
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
    return attend_group(c, g->prefix, layer, ws, g->gave_up, (cudaStream_t)stream);
} catch (...) {   // no exception leaves a C entry
    set_error("kv_group_attend: out of host memory");
    return -1;
}

}  // extern "C"
