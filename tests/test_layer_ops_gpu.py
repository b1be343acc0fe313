"""The single ops for callers that drive layers themselves, against plain
64-bit forms: rotary positions, token scores, attention over a cache (window,
sinks, rings) and attention of a batch that shares a prefix.

Tolerances. One rounding to bf16 is off by at most 2^-8 of the value, one to
f32 by 2^-24. Rotary: cosines and sines in f32 are off by at most 2^-22
(argument rounding pi 2^-25, function 2^-23), with two product roundings:
(|a| + |b|) mag 2^-21 in all, then the output's rounding. Attention: weights
rounded to bf16 over the sum of the same rounded weights move the normalised
weights by at most 2 * 2^-8; a score of D products in f32 is off by (D + 4)
2^-24 of sum |q k|, which enters a weight's exponent twice (weight and sum);
f32 accumulation adds 2^-14 for up to 2^10 sequential terms. Scores: sums of
at most V/128 + 64 sequential f32 terms, each off by 2^-21 of itself."""
import ctypes as C
import math
import threading

import numpy as np
import pytest
import torch

from mlxd_b200 import cuda
from tests.helpers import bf16_to_f32, f32_to_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    cuda.init(0)
    yield


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(20)


def rand(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def here():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------ rotary positions

def rope_angles(c, pos):
    """[n][pairs] angles in 64 bits and the magnitude, pair by pair."""
    out, mag, d = [], 1.0, c.dims
    for i in range(d // 2):
        w = float(c.theta) ** (-2.0 * i / d)
        f = float(c.factor)
        if c.scaling == cuda.ROPE_LINEAR:
            w /= f
        elif c.scaling == cuda.ROPE_LLAMA3:
            wl = 2 * math.pi / w
            if wl > c.orig_max / c.lo:
                w /= f
            elif wl > c.orig_max / c.hi:
                s = (c.orig_max / wl - c.lo) / (c.hi - c.lo)
                w = (1 - s) * w / f + s * w
        elif c.scaling == cuda.ROPE_YARN:
            at = lambda t: d * math.log(c.orig_max / (t * 2 * math.pi)) / (2 * math.log(c.theta))  # noqa: E731
            a, b = max(math.floor(at(c.hi)), 0), min(math.ceil(at(c.lo)), d - 1)
            r = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            w = r * w / f + (1 - r) * w
            mag = c.magnitude or 0.1 * math.log(f) + 1
        out.append(w)
    w = torch.tensor(out, dtype=torch.float64, device="cuda")
    return pos.double()[:, None] * w, mag


def rope_check(y, x, c, pos):
    d = c.dims
    ang, mag = rope_angles(c, pos)
    co, si = torch.cos(ang)[:, None] * mag, torch.sin(ang)[:, None] * mag
    r = x[..., :d].double()
    a, b = (r[..., 0::2], r[..., 1::2]) if c.interleaved else (r[..., :d // 2], r[..., d // 2:])
    g = y[..., :d].double()
    ga, gb = (g[..., 0::2], g[..., 1::2]) if c.interleaved else (g[..., :d // 2], g[..., d // 2:])
    half = 2.0 ** -8 if y.dtype == torch.bfloat16 else 2.0 ** -24
    slack = (a.abs() + b.abs()) * mag * 2.0 ** -21
    for got, want in ((ga, a * co - b * si), (gb, a * si + b * co)):
        assert bool(((got - want).abs() <= slack + half * (want.abs() + slack)).all())
    assert torch.equal(y[..., d:], x[..., d:])


def rope_call(x, c, pos, y, per_token=True):
    dt = cuda.BF16 if x.dtype == torch.bfloat16 else cuda.F32
    n, heads, D = x.shape
    cuda.check(cuda.lib().mlxd_cuda_rope(x.data_ptr(), dt, n, heads, D, x.stride(0), x.stride(1), C.byref(c),
                                         pos.data_ptr() if per_token else None, 0 if per_token else int(pos[0]),
                                         y.data_ptr(), y.stride(0), y.stride(1), here()), "rope")


SCALED = [dict(), dict(scaling=cuda.ROPE_LINEAR, factor=4.0),
          dict(scaling=cuda.ROPE_LLAMA3, factor=8.0, lo=1.0, hi=4.0, orig_max=8192),
          dict(scaling=cuda.ROPE_YARN, factor=16.0, lo=1.0, hi=32.0, orig_max=4096),
          dict(scaling=cuda.ROPE_YARN, factor=2.5, lo=2.0, hi=8.0, orig_max=512, magnitude=1.5)]


@pytest.mark.parametrize("scaled", SCALED, ids=["default", "linear", "llama3", "yarn", "yarn-mag"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,heads,D,dims", [(1, 1, 2, 2), (1, 40, 128, 128), (3, 5, 80, 40), (7, 2, 96, 24),
                                            (130, 9, 64, 64), (33, 3, 256, 256), (5, 3, 18, 6), (2, 72, 128, 64)])
def test_rope(gen, n, heads, D, dims, dtype, inter, scaled):
    x = rand(gen, n, heads, D, dtype=dtype)
    c = cuda.rope_config(1e4, dims, interleaved=inter, **scaled)
    pos = torch.randint(0, 200000, (n,), device="cuda", generator=gen).to(torch.int32)
    y = torch.full_like(x, 7)
    rope_call(x, c, pos, y)
    rope_check(y, x, c, pos)
    run = torch.arange(4091, 4091 + n, device="cuda", dtype=torch.int32)
    rope_call(x, c, run, y, per_token=False)
    rope_check(y, x, c, run)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("off,pad", [(0, 8), (1, 3), (4, 0), (8, 24)])
@pytest.mark.parametrize("inter", [False, True])
def test_rope_strides_and_alignment(gen, dtype, off, pad, inter):
    """Heads inside wider rows at any element offset, transposed output, guard elements untouched."""
    n, heads, D = 6, 5, 64
    base = rand(gen, n, heads * D + pad + off, dtype=dtype)
    x = base[:, off:off + heads * D].unflatten(1, (heads, D))
    out = torch.full((heads, n, D + pad), 3.0, device="cuda", dtype=dtype)   # [heads][n][..]: a cache's row order
    y = out[:, :, :D].transpose(0, 1)
    c = cuda.rope_config(1e6, 48, interleaved=inter)
    pos = torch.arange(100, 100 + n, device="cuda", dtype=torch.int32)
    rope_call(x, c, pos, y)
    rope_check(y, x, c, pos)
    assert bool((out[:, :, D:] == 3).all())


@pytest.mark.parametrize("n,heads,D,dims,off", [(2368, 70, 256, 32, 1), (2400, 72, 256, 0, 1), (600, 300, 256, 16, 1),
                                                (1200, 1100, 64, 64, 1), (1184, 33000, 8, 0, 0)])
def test_rope_many_heads_and_tokens(gen, n, heads, D, dims, off):
    """More (token, head, feature) items than one CTA takes of several tokens."""
    x = rand(gen, n * heads * D + off)[off:].view(n, heads, D)
    y = torch.full((n + 2, heads, D), 3.0, device="cuda", dtype=x.dtype)
    pos = torch.arange(5, 5 + n, device="cuda", dtype=torch.int32)
    c = cuda.rope_config(1e4, dims)
    rope_call(x, c, pos, y[1:-1])
    for i in range(0, n, 400):
        rope_check(y[1 + i:1 + min(i + 400, n)], x[i:i + 400], c, pos[i:i + 400])
    assert bool((y[0] == 3).all()) and bool((y[-1] == 3).all())


def test_rope_from_a_thread_without_a_context(gen):
    """The first CUDA call of a thread."""
    x = rand(gen, 9, 4, 64)
    y, c = torch.empty_like(x), cuda.rope_config(1e4, 64)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    args = (x.data_ptr(), cuda.BF16, 9, 4, 64, 256, 64, C.byref(c), pos.data_ptr(), 0, y.data_ptr(), 256, 64, None)
    rc = []
    t = threading.Thread(target=lambda: rc.append(cuda.lib().mlxd_cuda_rope(*args)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert rc == [0]
    rope_check(y, x, c, pos)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dims", [0, 20, 64])
def test_rope_in_place(gen, dtype, dims):
    x = rand(gen, 19, 6, 64, dtype=dtype)
    c = cuda.rope_config(1e4, dims)
    pos = torch.arange(0, 19, device="cuda", dtype=torch.int32)
    y = x.clone()
    rope_call(y, c, pos, y)
    rope_check(y, x, c, pos)


def test_rope_extreme_positions(gen):
    """Angles stay exact at the ends of the int32 range, and position 0 is the identity."""
    x = rand(gen, 5, 2, 128, dtype=torch.float32)
    c = cuda.rope_config(5e5, 128)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, 0, 1 << 24, -77], dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    rope_call(x, c, pos, y)
    rope_check(y, x, c, pos)
    assert torch.equal(y[2], x[2])


def test_rope_matches_model_table(gen):
    """The model path's own rule at the positions its f32 angles still hold (|angle| < 64: they are off by
    at most 64 * 2^-23, and its table is the f32 cosine of that)."""
    x = rand(gen, 64, 4, 64)
    c = cuda.rope_config(5e5, 64, scaling=cuda.ROPE_LLAMA3, factor=8.0, lo=1.0, hi=4.0, orig_max=8192)
    got = cuda.rope(x.view(torch.int16).cpu().numpy().view(np.uint16), c, 0)
    ang, _ = rope_angles(c, torch.arange(64, device="cuda"))
    co, si = (f(ang.float())[:, None] for f in (torch.cos, torch.sin))
    a, b = x[..., :32].float(), x[..., 32:].float()
    want = torch.cat((a * co - b * si, a * si + b * co), -1).cpu().numpy()
    bound = np.abs(want) * 2.0 ** -8 + 2.0 ** -15 * np.abs(x.float().cpu().numpy()).max()
    assert np.all(np.abs(bf16_to_f32(got) - want) <= bound)


# ------------------------------------------------------------------ token scores

def scores_call(x, targets, top, V=None, null=()):
    rows = x.shape[0]
    V = x.shape[1] if V is None else V
    o = dict(lp=torch.full((rows,), 9.0, device="cuda"), ent=torch.full((rows,), 9.0, device="cuda"),
             ids=torch.full((rows, top), -5, dtype=torch.int32, device="cuda"),
             tlp=torch.full((rows, top), 9.0, device="cuda"))
    p = {k: None if k in null else v.data_ptr() for k, v in o.items()}
    cuda.check(cuda.lib().mlxd_cuda_token_scores(x.data_ptr(), cuda.BF16 if x.dtype == torch.bfloat16 else cuda.F32,
                                                 rows, V, x.stride(0), targets.data_ptr(), top, p["lp"], p["ent"],
                                                 p["ids"], p["tlp"], here()), "token_scores")
    return o


def scores_check(o, x, targets, top):
    """Rows with a finite maximum."""
    V = x.shape[1]
    xd = x.double()
    m = xd.amax(1, keepdim=True)
    z = xd - m
    e = torch.exp(z)
    rest = e.scatter(1, xd.argmax(1, keepdim=True), 0.0).sum(1, keepdim=True)   # S - 1
    S = rest + 1
    logp = z - torch.log1p(rest)
    W = torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True)
    H = (torch.log1p(rest) - W / S)[:, 0]
    rel = (V / 128 + 64) * 2.0 ** -24 + 2.0 ** -21
    # the relative part counts the sum without the maximum's own term, which is what is accumulated
    tol = lambda v: (rel * rest / S + 2.0 ** -23 * v.abs()) + 1e-30  # noqa: E731
    want = logp.gather(1, targets.long()[:, None])[:, 0]
    near = torch.isfinite(want)
    assert bool((torch.isfinite(o["lp"]) == near).all())
    zt = z.gather(1, targets.long()[:, None]).abs()[:, 0]
    lim = (tol(want[:, None])[:, 0] + 2.0 ** -23 * zt)
    assert bool(((o["lp"].double() - want).abs()[near] <= lim[near]).all())
    wlim = rel * (rest / S + 2 * (W / S).abs())[:, 0] + 2.0 ** -23 * H.abs() + 1e-30
    assert bool(((o["ent"].double() - H).abs() <= wlim).all()), ((o["ent"].double() - H).abs() / wlim).max()
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(o["ids"].long(), order)
    wt = logp.gather(1, order)
    fin = torch.isfinite(wt)
    d = (o["tlp"].double() - wt).abs()
    assert bool((d[fin] <= (tol(wt) + 2.0 ** -23 * z.gather(1, order).abs())[fin]).all())
    assert bool((o["tlp"][~fin] == -math.inf).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,top,pad", [(1, 1, 1, 0), (3, 2, 2, 0), (1, 31, 5, 0), (2, 257, 32, 1),
                                            (5, 1000, 0, 0), (4, 4097, 1, 3), (1, 32768, 20, 0), (9, 50257, 20, 7),
                                            (1, 151936, 5, 0), (2, 151936, 32, 8), (40, 12345, 8, 0),
                                            (300, 2049, 3, 1), (17, 128256, 20, 0)])
def test_scores(gen, rows, V, top, pad, dtype):
    x = rand(gen, rows, V + pad, dtype=dtype, scale=3.0)[:, :V]
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen).to(torch.int32)
    scores_check(scores_call(x, t, top), x, t, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [600, 20011])
@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "few", "masked", "one", "zeros", "huge"])
def test_scores_hard_rows(gen, V, kind, dtype):
    """Ties over the whole row, sorted rows, masks that leave a few tokens or one, signed zeros, far magnitudes."""
    rows, top = 3, 32
    x = rand(gen, rows, V, dtype=torch.float32, scale=3.0)
    if kind == "equal":
        x = torch.full_like(x, -2.5)
    elif kind in ("ascending", "descending"):
        x = torch.sort(x, dim=1, descending=kind == "descending").values
    elif kind == "few":
        x = torch.round(x)
    elif kind == "masked":
        x[:, torch.rand(V, device="cuda", generator=gen) < 0.99] = -math.inf
        x[:, V // 2] = 1.0
    elif kind == "one":
        x[:] = -math.inf
        x[:, V - 1] = -3.0
    elif kind == "zeros":
        x = torch.where(x > 0, 0.0, -0.0)
    elif kind == "huge":
        x = x * 1e30
    x = x.to(dtype)
    t = torch.tensor([0, V // 2, V - 1], dtype=torch.int32, device="cuda")
    o = scores_call(x, t, top)
    if kind == "one":
        assert o["lp"].tolist() == [-math.inf, -math.inf, 0.0] and o["ent"].tolist() == [0.0] * 3
        assert o["ids"][0].tolist() == [V - 1] + list(range(31)) and o["tlp"][0, 0] == 0
        return
    scores_check(o, x, t, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [2, 80])
@pytest.mark.parametrize("kind", ["late", "rising", "strided", "few late", "gaps"])
def test_scores_rows_ordered_against_the_scan(gen, kind, rows, dtype):
    """Rows whose largest logits come late, rise along the row, lie where a few threads read, or are the only ones."""
    V = 70001
    x = rand(gen, rows, V, dtype=torch.float32)
    at = torch.arange(V, device="cuda")
    if kind == "late":
        x[:, :V // 3] = -math.inf
        x -= 700.0
    elif kind == "rising":
        x += at * 1e-3
    elif kind == "strided":
        n = 8 if dtype == torch.bfloat16 else 4
        x[:, (at // n) % 256 < 3] += 9.0
    elif kind == "gaps":        # threads that see nothing above -inf until late, then a rising rest
        n = 8 if dtype == torch.bfloat16 else 4
        x[:, ((at // n) % 256 % 4 < 3) & (at < V // 2)] = -math.inf
        x += at * 1e-4
    else:
        x[:, :V - 40] = -math.inf
    x = x.to(dtype)
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen).to(torch.int32)
    scores_check(scores_call(x, t, 20), x, t, 20)


@pytest.mark.parametrize("kind", ["random", "rising", "ties", "strided"])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_scores_repeat_bit_for_bit(gen, kind, rows):
    """Whatever order the threads meet the largest logits in (and when they are too many to list)."""
    V = 60013
    x = rand(gen, rows, V, dtype=torch.float32, scale=3.0)
    at = torch.arange(V, device="cuda")
    if kind == "rising":
        x += at * 1e-3
    elif kind == "ties":
        x = torch.round(x)
    elif kind == "strided":
        x[:, (at // 4) % 256 < 3] += 9.0
    t = torch.randint(0, V, (rows,), device="cuda", generator=gen).to(torch.int32)
    first = scores_call(x, t, 20)
    for _ in range(20):
        again = scores_call(x, t, 20)
        for k in first:
            assert torch.equal(again[k], first[k]), k


def test_scores_peaked_rows_keep_their_small_terms(gen):
    """A row whose other tokens hold 1e-12 of the mass: entropy and logprob to f32 precision of themselves."""
    V = 3001
    x = torch.zeros(2, V, device="cuda")
    x[:, 77] = 35.0
    x[1, 500] = 20.0
    t = torch.tensor([77, 77], dtype=torch.int32, device="cuda")
    scores_check(scores_call(x, t, 2), x, t, 2)


def test_scores_rows_without_a_distribution(gen):
    V, nan, inf = 700, math.nan, math.inf
    x = rand(gen, 4, V, dtype=torch.float32)
    x[0] = -inf
    x[1, 5] = inf
    x[2, 600] = nan
    t = torch.tensor([3, 5, 3, 3], dtype=torch.int32, device="cuda")
    o = scores_call(x, t, 4)
    assert o["lp"][0] == -inf and o["ent"][0] == 0 and o["ids"][0].tolist() == [0, 1, 2, 3]
    assert o["tlp"][0].tolist() == [-inf] * 4
    for r in (1, 2):
        assert o["lp"][r].isnan() and o["ent"][r].isnan() and bool(o["tlp"][r].isnan().all())
    assert o["ids"][1, 0] == 5 and 600 not in o["ids"][2].tolist()
    x[0] = nan
    o = scores_call(x[:1], t[:1], 3)
    assert o["lp"][0].isnan() and o["ids"][0].tolist() == [0, 1, 2]
    scores_check({k: v[3:] for k, v in scores_call(x, t, 4).items()}, x[3:], t[3:], 4)


def test_scores_targets_outside_and_missing_outputs(gen):
    x = rand(gen, 3, 99)
    t = torch.tensor([-1, 99, 98], dtype=torch.int32, device="cuda")
    o = scores_call(x, t, 2)
    assert o["lp"][0].isnan() and o["lp"][1].isnan() and o["lp"][2].isfinite()
    for k in ("lp", "ent", "ids", "tlp"):
        part = scores_call(x, t, 2, null=(k,))
        for j in o:
            want = torch.full_like(o[j], -5 if j == "ids" else 9.0) if j == k else o[j]
            assert torch.equal(part[j].nan_to_num(7), want.nan_to_num(7)), (k, j)


def test_scores_host_wrapper_and_sampler_agree():
    """The sampled token's logprob is the score of that token (both off by at most 2^-20 + 2^-23 |lp|)."""
    rng = np.random.default_rng(3)
    x = f32_to_bf16(rng.standard_normal(32768).astype(np.float32) * 3)
    tok, lp, _ = cuda.sample(x, cuda.sampling(temperature=0.0))
    s, _, ids, top = cuda.token_scores(x[None], [tok], 3)
    assert ids[0, 0] == tok and top[0, 0] == s[0]
    assert abs(s[0] - lp) <= 2.0 ** -15 * 2 + 2.0 ** -22 * abs(lp)


# ------------------------------------------------------------------ attention

def attn_tolerance(w, v, z_abs, out):
    """w [.., keys] exact weights, v [keys, D], z_abs: largest scale * sum |q k| of a row."""
    A = w @ v.abs()
    D = v.shape[-1]
    delta = (D + 4) * 2.0 ** -24 * z_abs + 2.0 ** -20
    return A * (2.0 ** -7 + 2 * delta + 2.0 ** -14) + out.abs() * 2.0 ** -8 + 1e-30


def attn_row(q, k, v, hide, scale):
    """One head: q [n, D], k/v [keys, D], hide [n, keys]: (out, tolerance) in 64 bits; rows that see nothing are 0."""
    q, k, v = q.double(), k.double(), v.double()
    k = torch.where(hide.all(0)[:, None], 0.0, k)
    v = torch.where(hide.all(0)[:, None], 0.0, v)
    z = (q @ k.T * scale).masked_fill(hide, -math.inf)
    w = torch.softmax(z, -1).nan_to_num(0.0)
    out = w @ v
    za = (q.abs() @ k.abs().T * scale).masked_fill(hide, 0).amax(-1, keepdim=True)
    return out, attn_tolerance(w, v, za, out)


def seen(qpos, kpos, window, sinks):
    near = (qpos - kpos < window) | (kpos < sinks) if window else torch.ones_like(qpos - kpos, dtype=torch.bool)
    return (kpos <= qpos) & near


class Cache:
    """Rows of every position in host order beside the library's cache; unwritten slots hold NaN bits."""

    def __init__(self, g, hkv, D, cap, total, window=0, sinks=0, layers=2, layer=1):
        self.kv = cuda.KVCache.shaped(layers, hkv, D, cap, window=window, sinks=sinks)
        self.layer, self.hkv, self.D = layer, hkv, D
        bad = torch.full((hkv, cap, D), math.nan, device="cuda", dtype=torch.bfloat16)
        ring = cap - sinks
        for l in range(layers):
            if sinks:
                self.kv.write(l, 0, bad[:, :sinks].contiguous(), bad[:, :sinks].contiguous())
            self.kv.write(l, sinks, bad[:, :ring].contiguous(), bad[:, :ring].contiguous())
        self.k, self.v = rand(g, hkv, total, D), rand(g, hkv, total, D)
        a = 0
        while a < total:
            step = min(total - a, sinks - a if a < sinks else ring)
            self.kv.write(layer, a, self.k[:, a:a + step].contiguous(), self.v[:, a:a + step].contiguous())
            a += step

    def attend(self, q, pos, cfg, out=None, stream=None):
        out = torch.empty_like(q) if out is None else out
        ws = torch.empty(cuda.attn_workspace_bytes(self.D), dtype=torch.uint8, device="cuda")
        cuda.check(cuda.lib().mlxd_cuda_kv_attend(self.kv.kv, self.layer, q.data_ptr(), q.stride(0), q.shape[0], pos,
                                                  C.byref(cfg), out.data_ptr(), out.stride(0), ws.data_ptr(),
                                                  ws.numel(), here() if stream is None else stream), "kv_attend")
        self.ws = ws
        return out

    def check(self, out, q, pos, window=0, sinks=0, scale=None, heads=None):
        n, hq, D = q.shape
        rep = hq // self.hkv
        scale = scale or D ** -0.5
        qpos = torch.arange(pos, pos + n, device="cuda")[:, None]
        hide = ~seen(qpos, torch.arange(pos + n, device="cuda")[None, :], window, sinks)
        assert bool(torch.isfinite(out).all())
        for h in heads or range(hq):
            want, tol = attn_row(q[:, h], self.k[h // rep, :pos + n], self.v[h // rep, :pos + n], hide, scale)
            err = (out[:, h].double() - want).abs()
            assert bool((err <= tol).all()), (h, float((err / tol).max()))


@pytest.mark.parametrize("hkv,rep,D", [(2, 4, 128), (1, 8, 64), (3, 1, 80), (2, 7, 96), (1, 32, 128), (2, 2, 16),
                                       (1, 3, 8), (2, 5, 256), (2, 16, 64), (1, 2, 136), (1, 4, 192)])
@pytest.mark.parametrize("n,pos", [(1, 0), (1, 63), (1, 300), (1, 2191), (2, 0), (5, 127), (33, 96), (130, 0),
                                   (300, 517)])
def test_attend(gen, n, pos, hkv, rep, D):
    """Lengths from one token up, odd sizes, every head layout; the rows behind the last position hold NaN."""
    c = Cache(gen, hkv, D, pos + n + 37, pos + n)
    q = rand(gen, n, hkv * rep, D, scale=1.5)
    c.check(c.attend(q, pos, cuda.attn_config(hkv * rep)), q, pos, heads=sorted({0, rep - 1, hkv * rep - 1}))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,pos,window,sinks,slack", [(1, 50, 1, 0, 0), (1, 50, 1, 2, 0), (1, 1000, 24, 4, 3),
                                                      (1, 9000, 4096, 4, 0), (3, 700, 65, 1, 0), (16, 4000, 500, 7, 1),
                                                      (64, 640, 128, 0, 0), (200, 1999, 300, 130, 5), (9, 0, 40, 4, 0),
                                                      (100, 30, 50, 16, 0), (257, 5000, 1024, 4, 77)])
def test_attend_ring(gen, n, pos, window, sinks, slack, D):
    """Wrapped and unwrapped rings that keep the sinks, at the smallest capacity that holds the window; the rows of
    other positions are overwritten or NaN."""
    c = Cache(gen, 2, D, sinks + window + n - 1 + slack, pos + n, window=window, sinks=sinks)
    q = rand(gen, n, 8, D, scale=1.5)
    c.check(c.attend(q, pos, cuda.attn_config(8, window=window, sinks=sinks)), q, pos, window, sinks, heads=[0, 5])
    if window > 10 and sinks > 1:       # narrower than the ring was made for
        o = c.attend(q, pos, cuda.attn_config(8, window=window - 9, sinks=sinks - 1))
        c.check(o, q, pos, window - 9, sinks - 1, heads=[3])


def test_attend_long_single_token(gen):
    for window, sinks, cap in ((0, 0, 33000), (30000, 4, 33004)):
        c = Cache(gen, 8, 128, cap, 32768, window=window, sinks=sinks, layers=1, layer=0)
        q = rand(gen, 1, 32, 128, scale=1.5)
        c.check(c.attend(q, 32767, cuda.attn_config(32, window=window, sinks=sinks)), q, 32767, window, sinks,
                heads=[0, 13, 31])


def test_attend_large_chunk(gen):
    c = Cache(gen, 2, 128, 3000, 3000, layers=1, layer=0)
    q = rand(gen, 1777, 16, 128, scale=1.5)
    c.check(c.attend(q, 1223, cuda.attn_config(16)), q, 1223, heads=[0, 9, 15])


def test_attend_wide_heads_long(gen):
    """Head dim 256: a single token over a long cache (split and joined), a chunk in several launches' worth of rows."""
    c = Cache(gen, 2, 256, 9000, 9000, layers=1, layer=0)
    q = rand(gen, 1, 16, 256, scale=1.5)
    c.check(c.attend(q, 8999, cuda.attn_config(16)), q, 8999, heads=[0, 9])
    q = rand(gen, 700, 16, 256, scale=1.5)
    c.check(c.attend(q, 5000, cuda.attn_config(16)), q, 5000, heads=[3, 15])


@pytest.mark.parametrize("n", [1, 40, 200])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_strided_rows_and_scale(gen, n, D):
    """q inside a fused projection's rows, out inside wider rows whose other elements stay."""
    c = Cache(gen, 2, D, 400, 100 + n)
    wide = rand(gen, n, 12 * D, scale=1.0)
    q = wide[:, :8 * D].unflatten(1, (8, D))
    o = torch.full((n + 1, 9 * D + 8), 5.0, device="cuda", dtype=torch.bfloat16)
    out = o[:n, :8 * D].unflatten(1, (8, D))
    c.attend(q, 100, cuda.attn_config(8, scale=0.37), out=out)
    c.check(out, q, 100, scale=0.37)
    assert bool((o[n:] == 5).all()) and bool((o[:, 8 * D:] == 5).all())


@pytest.mark.parametrize("n", [1, 150])
def test_attend_extreme_scores(gen, n):
    """Scores of +-2000 (all weight on one key, underflow elsewhere) and identical keys."""
    c = Cache(gen, 1, 64, 512, 300 + n)
    q = rand(gen, n, 4, 64, scale=60.0)
    o = c.attend(q, 300, cuda.attn_config(4))
    assert bool(torch.isfinite(o).all())
    c2 = Cache(gen, 1, 64, 512, 300 + n)
    same = c2.k[:, :1].expand(-1, 300 + n, -1).contiguous()
    c2.kv.write(c2.layer, 0, same, c2.v)
    c2.k = same
    q = rand(gen, n, 4, 64)
    c2.check(c2.attend(q, 300, cuda.attn_config(4)), q, 300)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,total", [(1, 100), (1, 9000), (3, 500), (40, 3000), (300, 700)])
def test_attend_nan_stays_in_its_row(gen, n, total, D):
    """A query of NaN gives NaN, its neighbours what they would give without it."""
    c = Cache(gen, 1, D, total, total)
    q = rand(gen, n, 4, D)
    clean = c.attend(q, total - n, cuda.attn_config(4))
    q[n // 2, 2] = math.nan
    out = c.attend(q, total - n, cuda.attn_config(4))
    assert bool(out[n // 2, 2].isnan().all())
    out[n // 2, 2] = clean[n // 2, 2]
    assert torch.equal(out, clean)


def test_attend_other_stream_and_graph(gen):
    """On a stream of its own, and captured once and replayed with new inputs; a second captured call shares the
    workspace in stream order."""
    s = torch.cuda.Stream()
    c = Cache(gen, 8, 128, 2048, 1500)
    cfg, one = cuda.attn_config(32), cuda.attn_config(32, window=100, sinks=2)
    q, q1 = rand(gen, 200, 32, 128), rand(gen, 1, 32, 128)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first, first1 = c.attend(q, 1300, cfg), c.attend(q1, 1499, one)
        out, out1 = torch.zeros_like(q), torch.zeros_like(q1)
        ws = torch.empty(cuda.attn_workspace_bytes(128), dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            for qq, pos, cf, o in ((q, 1300, cfg, out), (q1, 1499, one, out1)):
                cuda.check(cuda.lib().mlxd_cuda_kv_attend(c.kv.kv, c.layer, qq.data_ptr(), qq.stride(0), qq.shape[0],
                                                          pos, C.byref(cf), o.data_ptr(), o.stride(0), ws.data_ptr(),
                                                          ws.numel(), here()), "kv_attend")
        g.replay()
    s.synchronize()
    assert torch.equal(out, first) and torch.equal(out1, first1)
    q.mul_(-0.5)
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    c.check(out, q, 1300, heads=[1, 30])


def test_attend_repeats_bit_for_bit(gen):
    c = Cache(gen, 8, 128, 9000, 8500)
    for n in (1, 3, 64, 300):
        q = rand(gen, n, 32, 128)
        a = c.attend(q, 8500 - n, cuda.attn_config(32))
        for _ in range(3):
            assert torch.equal(a, c.attend(q, 8500 - n, cuda.attn_config(32)))


def test_attend_refusals(gen):
    """Arguments that a cache cannot serve come back as -1 with a message and write nothing."""
    L = cuda.lib()
    c = Cache(gen, 2, 64, 40, 60, window=30, sinks=2)
    q, out = rand(gen, 8, 4, 64), torch.full((8, 4, 64), 5.0, device="cuda", dtype=torch.bfloat16)
    ws = torch.empty(cuda.attn_workspace_bytes(64), dtype=torch.uint8, device="cuda")

    def call(word, layer=1, n=1, pos=59, cfg=None, qp=q.data_ptr(), qs=256, op=out.data_ptr(), os=256,
             wp=ws.data_ptr(), wb=ws.numel(), **kw):
        cfg = cfg or cuda.attn_config(4, window=30, sinks=2)
        rc = L.mlxd_cuda_kv_attend(c.kv.kv, layer, qp, qs, n, pos, C.byref(cfg), op, os, wp, wb, None)
        assert rc == -1 and word in L.mlxd_cuda_last_error().decode(), L.mlxd_cuda_last_error()

    call("bad arguments", layer=2)
    call("bad arguments", layer=-1)
    call("bad arguments", n=-1)
    call("bad arguments", pos=-1)
    call("bad arguments", pos=2 ** 31 - 1)
    for cfg in (cuda.attn_config(0), cuda.attn_config(3), cuda.attn_config(4, window=-1), cuda.attn_config(4, sinks=-1),
                cuda.attn_config(4, scale=-1.0), cuda.attn_config(4, scale=math.nan)):
        call("bad attention parameters", cfg=cfg)
    call("not held", cfg=cuda.attn_config(4))                       # the whole past of a wrapped ring
    call("not held", cfg=cuda.attn_config(4, window=39))            # wider than the ring
    call("not held", n=10, pos=50, cfg=cuda.attn_config(4, window=30))
    call("sinks", cfg=cuda.attn_config(4, window=30, sinks=3))
    call("alignment", qs=255)
    call("alignment", qs=260)
    call("alignment", os=248)
    call("alignment", qp=q.data_ptr() + 2)
    call("workspace", wb=ws.numel() - 1)
    call("workspace", wp=ws.data_ptr() + 16)
    call("null pointer", qp=None)
    host = np.zeros((4096,), np.uint16)
    aligned = host.ctypes.data + (-host.ctypes.data) % 16
    call("not device memory", qp=aligned)
    call("null pointer", wp=None)
    torch.cuda.synchronize()
    assert bool((out == 5).all())
    flat = cuda.KVCache.shaped(1, 2, 64, 40)
    rc = L.mlxd_cuda_kv_attend(flat.kv, 0, q.data_ptr(), 256, 8, 33, C.byref(cuda.attn_config(4, window=8)),
                               out.data_ptr(), 256, ws.data_ptr(), ws.numel(), None)
    assert rc == -1 and b"not held" in L.mlxd_cuda_last_error()     # past the end of a cache that is no ring
    assert L.mlxd_cuda_kv_attend(flat.kv, 0, q.data_ptr(), 256, 0, 0, C.byref(cuda.attn_config(4)), out.data_ptr(),
                                 256, ws.data_ptr(), ws.numel(), None) == 0
    odd = lambda x=0, y=0, p=0: L.mlxd_cuda_rope(q.data_ptr() + x, cuda.BF16, 1, 4, 64, 256, 64, C.byref(  # noqa: E731
        cuda.rope_config(1e4, 64)), ws.data_ptr() + 256 + p, 0, out.data_ptr() + y, 256, 64, None)
    for kw in (dict(x=1), dict(y=1), dict(p=2)):
        assert odd(**kw) == -1 and b"not aligned" in L.mlxd_cuda_last_error()
    lg = lambda x=0, t=0, o=0: L.mlxd_cuda_token_scores(q.data_ptr() + x, cuda.F32, 1, 64, 64, ws.data_ptr() + t, 0,  # noqa: E731
                                                        out.data_ptr() + o, None, None, None, None)
    for kw in (dict(x=2), dict(t=1), dict(o=2)):
        assert lg(**kw) == -1 and b"not aligned" in L.mlxd_cuda_last_error()
    assert L.mlxd_cuda_rope(q.data_ptr(), cuda.BF16, 1, 4, 64, 256, 64, C.byref(cuda.rope_config(1e4, 64)), None, 0,
                            aligned, 256, 64, None) == -1
    assert b"not device memory" in L.mlxd_cuda_last_error()


def test_sink_cache_rows_and_model_refusal(gen):
    """kv_gather, kv_write and kv_read follow the ring that keeps the sinks; the model's calls refuse such caches."""
    hkv, D, cap, sinks, window, total = 2, 64, 20, 3, 10, 50
    c = Cache(gen, hkv, D, cap, total, window=window, sinks=sinks, layers=1, layer=0)
    L = cuda.lib()
    got = torch.empty(hkv, sinks, D, device="cuda", dtype=torch.bfloat16)
    cuda.check(L.mlxd_cuda_kv_gather(c.kv.kv, 0, 0, 0, sinks, got.data_ptr(), None), "gather")
    near = torch.empty(hkv, cap - sinks, D, device="cuda", dtype=torch.bfloat16)
    first = total - (cap - sinks)
    cuda.check(L.mlxd_cuda_kv_gather(c.kv.kv, 0, 1, first, cap - sinks, near.data_ptr(), None), "gather")
    torch.cuda.synchronize()
    assert torch.equal(got, c.k[:, :sinks]) and torch.equal(near, c.v[:, first:total])
    cuda.check(L.mlxd_cuda_kv_set_offset(c.kv.kv, total, None), "set_offset")
    rows = c.kv.read(0, value=True)
    want = torch.cat((c.v[:, :sinks], c.v[:, first:total]), 1).view(torch.int16).cpu().numpy().view(np.uint16)
    assert np.array_equal(rows, want)
    assert L.mlxd_cuda_kv_write(c.kv.kv, 0, 30, cap - sinks + 1, c.k.data_ptr(), c.v.data_ptr(), None) == -1
    cfg = cuda.synth_config(hidden=256, layers=1, n_heads=4, n_kv_heads=2, head_dim=64, inter=256, vocab=256, max_pos=64)
    m = cuda.Model(cfg, cuda.synth_host_tensors(cfg, seed=1))
    flat = cuda.KVCache.shaped(1, 2, 64, 32)
    for ids in ([1], [1, 2, 3]):
        with pytest.raises(cuda.CudaError, match="kv_create_shape"):
            m.forward(flat, ids)


# ------------------------------------------------------------------ shared prefix

class Group:
    def __init__(self, g, hkv, D, prefix, cap, seqs, tail, layers=2, layer=1):
        self.pre = Cache(g, hkv, D, cap, prefix, layers=layers, layer=layer) if prefix else None
        kv = self.pre.kv if prefix else cuda.KVCache.shaped(layers, hkv, D, cap)
        self.kv, self.layer, self.prefix, self.hkv, self.D, self.tail = kv, layer, prefix, hkv, D, tail
        self.k = self.pre.k if prefix else rand(g, hkv, 0, D)
        self.v = self.pre.v if prefix else rand(g, hkv, 0, D)
        self.g = cuda.KVGroup(kv, prefix, seqs, tail)
        self.tk, self.tv = rand(g, seqs, hkv, tail, D), rand(g, seqs, hkv, tail, D)
        nan = torch.full((hkv, tail, D), math.nan, device="cuda", dtype=torch.bfloat16)
        for l in range(layers):
            for i in range(seqs):
                self.g.write(l, i, 0, nan, nan)

    def fill(self, lens):
        for i, m in enumerate(lens):
            m = min(m, self.tail)
            if m > 0:
                self.g.write(self.layer, i, 0, self.tk[i, :, :m].contiguous(), self.tv[i, :, :m].contiguous())

    def attend(self, q, lens, cfg, out=None):
        out = torch.full_like(q, 5.0) if out is None else out
        ws = torch.empty(cuda.attn_workspace_bytes(self.D), dtype=torch.uint8, device="cuda")
        cuda.check(cuda.lib().mlxd_cuda_kv_group_attend(self.g.g, self.layer, q.data_ptr(), q.stride(0),
                                                        lens.data_ptr(), C.byref(cfg), out.data_ptr(), out.stride(0),
                                                        ws.data_ptr(), ws.numel(), here()), "kv_group_attend")
        self.ws = ws
        return out

    def check(self, out, q, lens, window=0, sinks=0, seqs=None):
        n, hq, D = q.shape
        rep = hq // self.hkv
        for i in seqs if seqs is not None else range(n):
            m = lens[i]
            if m < 0:
                assert bool((out[i] == 5).all())
                continue
            m = min(m, self.tail)
            for g in range(self.hkv):
                k = torch.cat((self.k[g, :self.prefix], self.tk[i, g, :m]))
                v = torch.cat((self.v[g, :self.prefix], self.tv[i, g, :m]))
                qpos = torch.full((rep, 1), self.prefix + m - 1, device="cuda")
                hide = ~seen(qpos, torch.arange(self.prefix + m, device="cuda")[None, :], window, sinks)
                if self.prefix + m == 0:
                    assert bool((out[i] == 0).all())
                    continue
                want, tol = attn_row(q[i, g * rep:(g + 1) * rep], k, v, hide, D ** -0.5)
                err = (out[i, g * rep:(g + 1) * rep].double() - want).abs()
                assert bool((err <= tol).all()), (i, g, float((err / tol).max()))


@pytest.mark.parametrize("hkv,rep,D", [(2, 4, 128), (1, 8, 64), (3, 1, 80), (2, 5, 256), (1, 32, 128), (4, 2, 16)])
@pytest.mark.parametrize("seqs,prefix,tail", [(1, 0, 1), (1, 1, 5), (3, 0, 70), (2, 300, 33), (8, 1025, 64),
                                              (37, 517, 130), (70, 64, 9)])
def test_shared_prefix(gen, hkv, rep, D, seqs, prefix, tail):
    """Ragged tails beside finished, empty and over-long ones; prefix rows behind its length and unwritten tail rows
    hold NaN."""
    t = Group(gen, hkv, D, prefix, prefix + 19, seqs, tail)
    lens = [int(v) for v in torch.randint(1, tail + 1, (seqs,), device="cuda", generator=gen)]
    if seqs > 2:
        lens[0], lens[1], lens[2] = 0, -1, tail + 3
    t.fill(lens)
    q = rand(gen, seqs, hkv * rep, D, scale=1.5)
    out = t.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), cuda.attn_config(hkv * rep))
    t.check(out, q, lens, seqs=sorted({0, 1, 2, seqs // 2, seqs - 1} & set(range(seqs))))


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (40, 0), (200, 4), (500, 600), (5000, 1)])
def test_shared_prefix_window(gen, window, sinks):
    """Windows that end in the tail, in the prefix and before it, sinks in the prefix and past it."""
    lens = [1, 60, 13, 0, 64, 37]
    t = Group(gen, 2, 128, 450, 450, 6, 64)
    t.fill(lens)
    q = rand(gen, 6, 8, 128, scale=1.5)
    out = t.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                   cuda.attn_config(8, window=window, sinks=sinks))
    t.check(out, q, lens, window, sinks)


def test_shared_prefix_sees_nothing(gen):
    """No prefix and empty tails: zero rows, finished rows left alone."""
    t = Group(gen, 2, 64, 0, 8, 4, 16)
    lens = [0, -3, 2, 0]
    t.fill(lens)
    q = rand(gen, 4, 4, 64)
    out = t.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), cuda.attn_config(4))
    t.check(out, q, lens)


def test_shared_prefix_many_sequences(gen):
    t = Group(gen, 8, 128, 3000, 3100, 64, 200, layers=1, layer=0)
    lens = [int(v) for v in torch.randint(1, 201, (64,), device="cuda", generator=gen)]
    t.fill(lens)
    q = rand(gen, 64, 32, 128, scale=1.5)
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = t.attend(q, ld, cuda.attn_config(32))
    t.check(out, q, lens, seqs=[0, 17, 31, 32, 63])
    for _ in range(3):
        assert torch.equal(out, t.attend(q, ld, cuda.attn_config(32)))


@pytest.mark.parametrize("D,seqs,tail", [(128, 24, 1500), (64, 20, 900), (96, 19, 700)])
def test_shared_prefix_long_tails(gen, D, seqs, tail):
    """Items that fill the SMs two or three times over: a cluster to a tail, some of them ended, empty or full."""
    t = Group(gen, 8, D, 1000, 1100, seqs, tail, layers=1, layer=0)
    lens = [int(v) for v in torch.randint(1, tail + 1, (seqs,), device="cuda", generator=gen)]
    lens[0], lens[1], lens[2], lens[3] = 0, -1, tail, 1
    t.fill(lens)
    q = rand(gen, seqs, 32, D, scale=1.5)
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = t.attend(q, ld, cuda.attn_config(32))
    t.check(out, q, lens, seqs=[0, 1, 2, 3, seqs - 1])
    for _ in range(5):
        again = t.attend(q, ld, cuda.attn_config(32))
        keep = [i for i in range(seqs) if lens[i] >= 0]
        assert torch.equal(out[keep], again[keep])


@pytest.mark.parametrize("hkv,D", [(160, 64), (200, 32)])
def test_attend_single_token_many_kv_heads(gen, hkv, D):
    c = Cache(gen, hkv, D, 700, 650, layers=1, layer=0)
    q = rand(gen, 1, hkv, D, scale=1.5)
    a = c.attend(q, 649, cuda.attn_config(hkv))
    c.check(a, q, 649, heads=[0, 1, hkv // 2, hkv - 1])
    assert torch.equal(a, c.attend(q, 649, cuda.attn_config(hkv)))


def test_attend_long_chunk_over_heads(gen):
    """More tiles than one wave, an odd number of them: every head's rows at their places."""
    c = Cache(gen, 5, 128, 2200, 2190, layers=1, layer=0)
    q = rand(gen, 1990, 20, 128, scale=1.5)
    a = c.attend(q, 200, cuda.attn_config(20))
    c.check(a, q, 200, heads=[0, 3, 4, 11, 19])
    assert torch.equal(a, c.attend(q, 200, cuda.attn_config(20)))


def test_group_decode_loop_in_a_graph(gen):
    """append + attend captured once and replayed with lengths that grow on the device, as a batched decode loop runs
    them; a finished sequence's rows stay."""
    seqs, hkv, D, prefix = 5, 2, 64, 150
    t = Group(gen, hkv, D, prefix, prefix, seqs, 12)
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    step = torch.tensor([1, 1, 0, 1, 1], dtype=torch.int32, device="cuda")
    lens[2] = -1
    kv = torch.zeros(seqs, 3 * hkv * D, device="cuda", dtype=torch.bfloat16)     # strided rows
    k, v = kv[:, :hkv * D], kv[:, 2 * hkv * D:]
    q = rand(gen, seqs, 8, D)
    out = torch.full_like(q, 5.0)
    ws = torch.empty(cuda.attn_workspace_bytes(D), dtype=torch.uint8, device="cuda")
    cfg, L = cuda.attn_config(8), cuda.lib()

    def body():
        lens.add_(step)
        cuda.check(L.mlxd_cuda_kv_group_append(t.g.g, t.layer, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                               lens.data_ptr(), here()), "append")
        cuda.check(L.mlxd_cuda_kv_group_attend(t.g.g, t.layer, q.data_ptr(), q.stride(0), lens.data_ptr(),
                                               C.byref(cfg), out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(),
                                               here()), "attend")

    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        body()
    for n in range(1, 13):
        k.copy_(t.tk[:, :, n - 1].reshape(seqs, -1))
        v.copy_(t.tv[:, :, n - 1].reshape(seqs, -1))
        g.replay()
        torch.cuda.synchronize()
        if n in (1, 5, 12):
            t.check(out, q, lens.tolist())
    g.replay()          # past the tails' capacity: nothing is written, the length counts as the capacity
    torch.cuda.synchronize()
    t.check(out, q, lens.tolist())


def test_group_refusals(gen):
    L = cuda.lib()
    kv = cuda.KVCache.shaped(1, 2, 64, 16)
    for args in ((17, 1, 4), (-1, 1, 4), (4, 0, 4), (4, 1, 0), (4, 1, 2 ** 31 - 1)):
        h = C.c_void_p(7)
        assert L.mlxd_cuda_kv_group_create(C.byref(h), kv.kv, *args) == -1 and h.value == 7
    t = Group(gen, 2, 64, 10, 16, 3, 4)
    x = rand(gen, 3, 4, 64)
    lens = torch.ones(3, dtype=torch.int32, device="cuda")
    ws = torch.empty(cuda.attn_workspace_bytes(64), dtype=torch.uint8, device="cuda")
    cfg = cuda.attn_config(4)
    att = lambda layer=0, c=cfg, ln=lens.data_ptr(), wb=ws.numel(): L.mlxd_cuda_kv_group_attend(  # noqa: E731
        t.g.g, layer, x.data_ptr(), 256, ln, C.byref(c), x.data_ptr(), 256, ws.data_ptr(), wb, None)
    for kw in (dict(layer=2), dict(c=cuda.attn_config(5)), dict(ln=None), dict(wb=8)):
        assert att(**kw) == -1 and L.mlxd_cuda_last_error() != b""
    app = lambda layer=0, ks=128, kp=x.data_ptr(): L.mlxd_cuda_kv_group_append(  # noqa: E731
        t.g.g, layer, kp, ks, x.data_ptr(), 128, lens.data_ptr(), None)
    for kw in (dict(layer=-1), dict(ks=120), dict(ks=132), dict(kp=x.data_ptr() + 2), dict(kp=None)):
        assert app(**kw) == -1
    for a in ((2, 0, 0, 1), (0, 3, 0, 1), (0, 0, 4, 1), (0, 0, 0, 5), (0, 0, -1, 1)):
        assert L.mlxd_cuda_kv_group_write(t.g.g, *a, x.data_ptr(), x.data_ptr(), None) == -1


# ------------------------------------------------------------------ together

def test_layer_driven_by_single_ops(gen):
    """One decoder layer's attention half, a chunk and then single tokens, as a caller runs it: projections, rotary
    positions into the cache's row order, kv_write, attention, output projection, lm_head and token scores."""
    H, hq, hkv, D, V, n = 256, 4, 2, 64, 512, 24
    cfg = cuda.synth_config(hidden=H, layers=1, n_heads=hq, n_kv_heads=hkv, head_dim=D, inter=256, vocab=V, max_pos=64)
    host = cuda.synth_host_tensors(cfg, seed=2, std=0.08)
    lin = lambda name: cuda.Linear(*(host[name + s] for s in (".weight", ".scales", ".biases")), 64)  # noqa: E731
    qkv = [lin("model.layers.0.self_attn.%s_proj" % c) for c in "qkv"]
    o, lm = lin("model.layers.0.self_attn.o_proj"), lin("lm_head")
    kv = cuda.KVCache.shaped(1, hkv, D, 64, window=16, sinks=2)
    ws = torch.empty(cuda.attn_workspace_bytes(D), dtype=torch.uint8, device="cuda")
    rc, ac, L = cuda.rope_config(1e6, D), cuda.attn_config(hq, window=16, sinks=2), cuda.lib()
    x = rand(gen, n, H)
    bits = lambda t: t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)  # noqa: E731
    dev = lambda a: torch.from_numpy(a.view(np.int16)).cuda().view(torch.bfloat16)  # noqa: E731
    att = []
    for a, b in ((0, 20), (20, 21), (21, 22), (22, 24)):
        m = b - a
        q, k, v = (dev(p(bits(x[a:b]))) for p in qkv)
        kr = torch.empty(hkv, m, D, device="cuda", dtype=torch.bfloat16)
        qr = torch.empty(m, hq, D, device="cuda", dtype=torch.bfloat16)
        pos = torch.arange(a, b, device="cuda", dtype=torch.int32)
        rope_call(q.unflatten(1, (hq, D)), rc, pos, qr, per_token=False)
        rope_call(k.unflatten(1, (hkv, D)), rc, pos, kr.transpose(0, 1))
        kv.write(0, a, kr, v.unflatten(1, (hkv, D)).transpose(0, 1).contiguous(), here())
        out = torch.empty_like(qr)
        cuda.check(L.mlxd_cuda_kv_attend(kv.kv, 0, qr.data_ptr(), qr.stride(0), m, a, C.byref(ac), out.data_ptr(),
                                         out.stride(0), ws.data_ptr(), ws.numel(), here()), "attend")
        att.append(out)
    att = torch.cat(att)
    logits = lm(o(bits(att.flatten(1))))
    lp, ent, ids, top = cuda.token_scores(logits, np.arange(n) % V, 4)

    # the same in 64 bits from the projections' own outputs
    q, k, v = (dev(p(bits(x))) for p in qkv)
    pos = torch.arange(n, device="cuda", dtype=torch.int32)
    q, k = (t.unflatten(1, (-1, D)) for t in (q, k))
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    rope_call(q, rc, pos, qr)
    rope_call(k, rc, pos, kr)
    rope_check(qr, q, rc, pos)
    hide = ~seen(pos[:, None], pos[None, :], 16, 2)
    for h in range(hq):
        want, tol = attn_row(qr[:, h], kr[:, h // 2], v.unflatten(1, (hkv, D))[:, h // 2], hide, D ** -0.5)
        assert bool(((att[:, h].double() - want).abs() <= tol).all())
    z = bf16_to_f32(logits).astype(np.float64)
    logp = z - np.log(np.exp(z).sum(1, keepdims=True))
    assert np.abs(lp - logp[np.arange(n), np.arange(n) % V]).max() <= 2.0 ** -18
    assert np.array_equal(ids, np.argsort(-z, axis=1, kind="stable")[:, :4])
    assert np.abs(ent + (np.exp(logp) * logp).sum(1)).max() <= 2.0 ** -16
