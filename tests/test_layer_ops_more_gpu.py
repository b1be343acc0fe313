"""Attention over a cache and of a shared prefix where the plain comparison is blind: every key is counted once, the
weights sum to one, maxima that rise along the keys, the bf16 pairs of few rows; against 64-bit forms.

Tolerances: a rounding to bf16 is off by at most 2^-8 of the value. Weights rounded to bf16 over the sum of the same
rounded weights move the normalised weights by at most 2 * 2^-8, weights held as two bf16 terms (8 + 8 bits and a sign)
by at most 2 * 2^-17. A score of D products in f32 is off by (D + 4) 2^-24 of sum |q k|, and enters exponents twice."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from mlxd_b200 import cuda
from tests.helpers import bf16_to_f32
from tests.test_layer_ops_gpu import Cache, Group, attn_row, rand, seen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    cuda.init(0)
    yield


@pytest.fixture
def gen():
    return torch.Generator(device="cuda").manual_seed(77)


def put(c, k=None, v=None):
    """Other rows for every position of a Cache, in runs that fit its ring."""
    total, ring, a = c.k.shape[1], c.kv.capacity() - c.sinks, 0
    c.k, c.v = c.k if k is None else k, c.v if v is None else v
    while a < total:
        step = min(total - a, c.sinks - a if a < c.sinks else ring)
        c.kv.write(c.layer, a, c.k[:, a:a + step].contiguous(), c.v[:, a:a + step].contiguous())
        a += step


def cache(g, hkv, D, cap, total, window=0, sinks=0):
    c = Cache(g, hkv, D, cap, total, window=window, sinks=sinks, layers=1, layer=0)
    c.sinks = sinks
    return c


# ------------------------------------------------------------------ every key once

def counts(hide, D, groups, i):
    """Values that are 1 in one feature (key j: feature j mod D groups, when that is among the i-th D), and what equal
    weights make of them: the feature's visible keys over all visible keys."""
    keys = hide.shape[1]
    at = torch.arange(keys, device="cuda") % (D * groups) - i * D
    v = torch.zeros(keys, D, device="cuda", dtype=torch.float64)
    j = torch.nonzero((at >= 0) & (at < D))[:, 0]
    v[j, at[j]] = 1.0
    see = (~hide).double()
    return v, see @ v / see.sum(1, keepdim=True)


def counted(got, want):
    """Equal scores make every weight exactly 1, so that sums are whole numbers: the division's rounding (2^-23) and the
    output's. A feature has at most 32 keys: one of them too few or too many is off by a 33rd."""
    return bool(((got.double() - want).abs() <= want * (2.0 ** -8 + 2.0 ** -22)).all())


@pytest.mark.parametrize("hkv,rep,D", [(8, 4, 128), (2, 7, 64), (1, 1, 80), (2, 12, 128), (2, 2, 256), (1, 12, 192),
                                       (1, 16, 16)])
@pytest.mark.parametrize("n,pos", [(1, 0), (1, 14), (1, 15), (1, 16), (1, 127), (1, 128), (1, 2191), (1, 4100),
                                   (1, 32767), (2, 1000), (3, 8190), (40, 2000), (150, 700), (700, 130)])
def test_attend_counts_every_key(gen, n, pos, hkv, rep, D):
    if n * rep * hkv * (pos + n) > 8e7:
        n = max(1, int(8e7 / (rep * hkv * (pos + n))))
    total = pos + n
    c = cache(gen, hkv, D, total + 5, total)
    q = torch.zeros(n, hkv * rep, D, device="cuda", dtype=torch.bfloat16)
    hide = ~seen(torch.arange(pos, total, device="cuda")[:, None], torch.arange(total, device="cuda")[None], 0, 0)
    groups = -(-total // (32 * D))
    for i in range(groups):
        v, want = counts(hide, D, groups, i)
        put(c, v=v.to(torch.bfloat16).expand(hkv, -1, -1).contiguous())
        out = c.attend(q, pos, cuda.attn_config(hkv * rep))
        assert counted(out, want[:, None]), i


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,pos,window,sinks,slack", [(1, 1000, 24, 4, 3), (1, 9000, 4096, 4, 0), (3, 700, 65, 1, 0),
                                                      (64, 640, 128, 0, 0), (200, 1999, 300, 130, 5), (9, 0, 40, 4, 0),
                                                      (257, 5000, 1024, 4, 77), (512, 3000, 700, 17, 0)])
def test_attend_ring_counts_every_key(gen, n, pos, window, sinks, slack, D):
    total = pos + n
    c = cache(gen, 2, D, sinks + window + n - 1 + slack, total, window, sinks)
    q = torch.zeros(n, 8, D, device="cuda", dtype=torch.bfloat16)
    hide = ~seen(torch.arange(pos, total, device="cuda")[:, None], torch.arange(total, device="cuda")[None], window, sinks)
    groups = -(-(window + sinks) // (31 * D))
    for i in range(groups):
        v, want = counts(hide, D, groups, i)
        put(c, v=v.to(torch.bfloat16).expand(2, -1, -1).contiguous())
        out = c.attend(q, pos, cuda.attn_config(8, window=window, sinks=sinks))
        assert counted(out, want[:, None]), i


@pytest.mark.parametrize("hkv,rep,D", [(2, 4, 128), (8, 4, 128), (1, 12, 64), (2, 3, 256)])
@pytest.mark.parametrize("seqs,prefix,tail", [(1, 1, 5), (3, 0, 300), (8, 1025, 64), (37, 517, 130), (24, 3000, 1000)])
def test_shared_prefix_counts_every_key(gen, hkv, rep, D, seqs, prefix, tail):
    t = Group(gen, hkv, D, prefix, prefix + 19, seqs, tail, layers=1, layer=0)
    lens = [int(x) for x in torch.randint(1, tail + 1, (seqs,), device="cuda", generator=gen)]
    lens[-1] = tail
    if seqs > 2:
        lens[1], lens[2] = 0 if prefix else 1, 17
    q = torch.zeros(seqs, hkv * rep, D, device="cuda", dtype=torch.bfloat16)
    groups = -(-(prefix + tail) // (32 * D))
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    hide = torch.arange(prefix + tail, device="cuda")[None] >= prefix + ld[:, None]
    for i in range(groups):
        v, want = counts(hide, D, groups, i)
        vb = v.to(torch.bfloat16).expand(hkv, -1, -1)
        if prefix:
            t.kv.write(0, 0, t.k, vb[:, :prefix].contiguous())
        t.tv = vb[None, :, prefix:].expand(seqs, -1, -1, -1)
        t.fill(lens)
        assert counted(t.attend(q, ld, cuda.attn_config(hkv * rep)), want[:, None]), i


# ------------------------------------------------------------------ maxima that rise along the keys

def rising(c, q, pos, scale, window=0, sinks=0):
    """Keys whose size grows along the positions, so that the rows' maxima jump again and again, and values that shrink
    by as much as the weights grow, so that what was summed before each jump counts in the result."""
    total = c.k.shape[1]
    g = 0.2 + 5.0 * torch.arange(total, device="cuda") / total
    sigma = q.double().pow(2).sum(-1).mean().sqrt() * scale      # of a score over keys of size 1
    k = (c.k.double() * g[:, None]).to(torch.bfloat16)
    v = (c.v.double() * torch.exp(3.0 * sigma * (g[-1] - g))[:, None]).to(torch.bfloat16)
    put(c, k, v)


@pytest.mark.parametrize("hkv,rep,D,n,pos", [(2, 8, 128, 1777, 1223), (2, 8, 64, 1777, 1223), (2, 8, 80, 1500, 900),
                                             (1, 32, 128, 300, 5000), (1, 32, 64, 300, 5000), (1, 16, 128, 40, 16000),
                                             (1, 16, 64, 41, 9001), (5, 4, 128, 1990, 200), (2, 4, 128, 1, 5000),
                                             (2, 4, 128, 2, 5000), (2, 4, 256, 40, 3000), (1, 12, 256, 1, 3000)])
def test_attend_rising_maxima(gen, hkv, rep, D, n, pos):
    c = cache(gen, hkv, D, pos + n + 3, pos + n)
    q = rand(gen, n, hkv * rep, D, scale=1.5)
    rising(c, q, pos, D ** -0.5)
    c.check(c.attend(q, pos, cuda.attn_config(hkv * rep)), q, pos, heads=sorted({0, rep - 1, hkv * rep - 1}))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,pos,window,sinks", [(512, 7680, 4096, 4), (1200, 6000, 1500, 4)])
def test_attend_ring_rising_maxima(gen, n, pos, window, sinks, D):
    c = cache(gen, 2, D, sinks + window + n - 1, pos + n, window, sinks)
    q = rand(gen, n, 16, D, scale=1.5)
    rising(c, q, pos, D ** -0.5)
    c.check(c.attend(q, pos, cuda.attn_config(16, window=window, sinks=sinks)), q, pos, window, sinks, heads=[0, 7, 9])


@pytest.mark.parametrize("n", [150, 1500])
def test_attend_extreme_scores_in_value(gen, n):
    """Scores of +-2000 over many tiles: what the 64-bit form gives, not finiteness alone."""
    c = cache(gen, 2, 64, 400 + n, 300 + n)
    q = rand(gen, n, 16, 64, scale=60.0)
    c.check(c.attend(q, 300, cuda.attn_config(16)), q, 300, heads=[0, 5, 15])


# ------------------------------------------------------------------ weights that sum to one

@pytest.mark.parametrize("hkv,rep,D,n,pos", [(2, 8, 128, 1777, 1223), (2, 8, 64, 700, 1223), (1, 32, 128, 300, 2000),
                                             (1, 16, 128, 40, 9000), (2, 4, 128, 1, 3001), (2, 16, 256, 30, 1000)])
def test_attend_of_equal_values_is_that_value(gen, hkv, rep, D, n, pos):
    """Whatever the weights are: f32 sums of the weights as they enter the product leave less than half a step."""
    c = cache(gen, hkv, D, pos + n, pos + n)
    q = rand(gen, n, hkv * rep, D, scale=1.5)
    total = pos + n
    # a few keys stand out by 4 to 7 bits late in the row, where the maximum in use stays an earlier one
    k = c.k.clone()
    k[:, ::301] *= 2.0
    one = rand(gen, hkv, 1, D).expand(-1, total, -1).contiguous()
    put(c, k, one)
    out = c.attend(q, pos, cuda.attn_config(hkv * rep))
    want = one[:, 0].repeat_interleave(rep, 0)
    assert torch.equal(out, want.expand(n, -1, -1))


# ------------------------------------------------------------------ few rows: weights as two bf16 terms

def pair_tolerance(q, k, v, hide, scale, out, parts):
    """Weights off by 2 * 2^-17, scores as above, and f32 sums of at most keys / (16 parts) + 64 steps, each off by 2^-22
    (a truncated product of 16 keys); then the output's rounding."""
    z = q.double() @ k.double().T * scale
    w = torch.softmax(z.masked_fill(hide, -math.inf), -1)
    za = (q.double().abs() @ k.double().abs().T * scale).masked_fill(hide, 0).amax(-1, keepdim=True)
    D, keys = k.shape[1], k.shape[0]
    delta = (D + 4) * 2.0 ** -24 * za + 2.0 ** -20
    return (w @ v.double().abs()) * (2.0 ** -16 + 2 * delta + (keys / (16 * parts) + 64) * 2.0 ** -22) + out.abs() * 2.0 ** -8


@pytest.mark.parametrize("hkv,rep,D,n,pos", [(8, 4, 128, 1, 300), (8, 4, 128, 1, 2191), (8, 4, 128, 1, 32767),
                                             (2, 8, 128, 1, 2191), (2, 8, 64, 1, 900), (1, 1, 80, 1, 500),
                                             (2, 4, 128, 2, 1500), (1, 8, 256, 1, 1000), (1, 3, 192, 2, 700)])
def test_attend_few_rows_keep_the_low_terms(gen, hkv, rep, D, n, pos):
    c = cache(gen, hkv, D, pos + n, pos + n)
    q = rand(gen, n, hkv * rep, D, scale=1.5)
    out = c.attend(q, pos, cuda.attn_config(hkv * rep))
    hide = ~seen(torch.arange(pos, pos + n, device="cuda")[:, None], torch.arange(pos + n, device="cuda")[None], 0, 0)
    for h in range(hkv * rep):
        k, v = c.k[h // rep], c.v[h // rep]
        want, _ = attn_row(q[:, h], k, v, hide, D ** -0.5)
        err = (out[:, h].double() - want).abs()
        tol = pair_tolerance(q[:, h], k, v, hide, D ** -0.5, want, 8)
        assert bool((err <= tol).all()), (h, float((err / tol).max()))


def test_shared_prefix_tails_keep_the_low_terms(gen):
    """No prefix: the tails' kernel alone."""
    t = Group(gen, 2, 128, 0, 8, 6, 700, layers=1, layer=0)
    lens = [1, 700, 33, 128, 499, 16]
    t.fill(lens)
    q = rand(gen, 6, 8, 128, scale=1.5)
    out = t.attend(q, torch.tensor(lens, dtype=torch.int32, device="cuda"), cuda.attn_config(8))
    for i, m in enumerate(lens):
        for h in range(8):
            k, v = t.tk[i, h // 4, :m], t.tv[i, h // 4, :m]
            hide = torch.zeros(1, m, dtype=torch.bool, device="cuda")
            want, _ = attn_row(q[i, h:h + 1], k, v, hide, 128 ** -0.5)
            err = (out[i, h:h + 1].double() - want).abs()
            assert bool((err <= pair_tolerance(q[i, h:h + 1], k, v, hide, 128 ** -0.5, want, 4)).all()), (i, h)


# ------------------------------------------------------------------ cache rows

def rows_refused(rc, word):
    msg = cuda.lib().mlxd_cuda_last_error().decode()
    assert rc == -1 and word in msg, (rc, msg)


def test_cache_rows_that_share_slots_are_refused(gen):
    """Rows from inside the sinks that reach round the whole ring: later positions would lie where the first do."""
    L, hkv, D, cap, sinks = cuda.lib(), 2, 64, 14, 4
    kv = cuda.KVCache.shaped(1, hkv, D, cap, window=10, sinks=sinks)
    x = rand(gen, hkv, cap, D)
    out = torch.full_like(x, 7.0)
    for pos, n in ((0, 14), (2, 12), (3, 11), (4, 10), (40, 10)):
        y = x[:, :n].contiguous()
        kv.write(0, pos, y, -y)
        o = torch.empty_like(y)
        cuda.check(L.mlxd_cuda_kv_gather(kv.kv, 0, 1, pos, n, o.data_ptr(), None), "gather")
        torch.cuda.synchronize()
        assert torch.equal(o, -y)
    for pos, n in ((1, 14), (2, 13), (3, 14), (4, 11)):
        rows_refused(L.mlxd_cuda_kv_write(kv.kv, 0, pos, n, x.data_ptr(), x.data_ptr(), None), "over a ring of 10 slots")
        rows_refused(L.mlxd_cuda_kv_gather(kv.kv, 0, 0, pos, n, out.data_ptr(), None), "over a ring of 10 slots")
    torch.cuda.synchronize()
    assert bool((out == 7).all())


def test_cache_rows_past_the_last_position_are_refused(gen):
    L = cuda.lib()
    x = rand(gen, 2, 8, 64)
    for kv in (cuda.KVCache.shaped(1, 2, 64, 14, window=10, sinks=4), cuda.KVCache.shaped(1, 2, 64, 9)):
        for pos, n in ((2 ** 31 - 1, 1), (2 ** 31 - 4, 8)):
            rows_refused(L.mlxd_cuda_kv_write(kv.kv, 0, pos, n, x.data_ptr(), x.data_ptr(), None), "bad arguments")
            rows_refused(L.mlxd_cuda_kv_gather(kv.kv, 0, 0, pos, n, x.data_ptr(), None), "bad arguments")


# ------------------------------------------------------------------ positions that a cache holds

def attend_rc(kv, layer, q, pos, window=0, sinks=0, stream=None):
    hq, D = q.shape[1:]
    out = torch.empty_like(q)
    ws = torch.empty(cuda.attn_workspace_bytes(D), dtype=torch.uint8, device="cuda")
    rc = cuda.lib().mlxd_cuda_kv_attend(kv.kv, layer, q.data_ptr(), q.stride(0), q.shape[0], pos,
                                        C.byref(cuda.attn_config(hq, window=window, sinks=sinks)), out.data_ptr(),
                                        out.stride(0), ws.data_ptr(), ws.numel(), stream)
    return rc, out, ws


def test_attend_refuses_rows_that_a_models_ring_has_overwritten(gen):
    cfg = cuda.synth_config(hidden=256, layers=2, n_heads=4, n_kv_heads=2, head_dim=64, inter=256, vocab=256,
                            family=cuda.MISTRAL, window=16, max_pos=128)
    m = cuda.Model(cfg, cuda.synth_host_tensors(cfg, seed=1))
    kv = m.new_kv(24)
    q = rand(gen, 2, 4, 64)
    rows_refused(attend_rc(kv, 0, q, 0)[0], "have not been written")
    m.forward(kv, list(range(9)))
    for t in range(3):
        m.forward(kv, [t])
    assert attend_rc(kv, 1, q, 10)[0] == 0 and attend_rc(kv, 0, q, 3)[0] == 0
    rows_refused(attend_rc(kv, 1, q, 11)[0], "have not been written")
    g, short = cuda.KVGroup(kv, 12, 2, 4), cuda.KVGroup(kv, 13, 2, 4)
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")

    def group(g):
        out = torch.empty_like(q)
        ws = torch.empty(cuda.attn_workspace_bytes(64), dtype=torch.uint8, device="cuda")
        return cuda.lib().mlxd_cuda_kv_group_attend(g.g, 1, q.data_ptr(), 256, lens.data_ptr(),
                                                    C.byref(cuda.attn_config(4)), out.data_ptr(), 256, ws.data_ptr(),
                                                    ws.numel(), None)

    assert group(g) == 0
    rows_refused(group(short), "have not been written")
    for a in range(12, 40, 7):
        m.forward(kv, list(range(7)))
    assert kv.offset() == 40
    rows_refused(attend_rc(kv, 1, q, 10)[0], "have been overwritten")
    rows_refused(attend_rc(kv, 0, q, 10, window=16)[0], "have been overwritten")
    rows_refused(attend_rc(kv, 0, q, 22, window=8)[0], "have been overwritten")        # positions 15 to 23, 16 is held
    assert attend_rc(kv, 0, q, 22, window=7)[0] == 0
    assert attend_rc(kv, 0, q, 38, window=16)[0] == 0
    rows_refused(group(g), "have been overwritten")
    h = C.c_void_p(7)
    rows_refused(cuda.lib().mlxd_cuda_kv_group_create(C.byref(h), kv.kv, 12, 2, 4), "has been overwritten")
    assert h.value == 7
    kv.reset()
    m.forward(kv, list(range(9)))
    assert attend_rc(kv, 1, q, 7)[0] == 0


@pytest.mark.parametrize("sinks", [0, 3])
def test_attend_takes_what_a_ring_holds_and_no_more(gen, sinks):
    """Runs appended, taken back and written again in any order without gaps: an accepted call's positions lie in their
    slots, and the run last written can always be attended to."""
    D, ring = 8, 13
    cap = sinks + ring
    kv = cuda.KVCache.shaped(1, 1, D, cap, window=5, sinks=sinks)
    r = torch.Generator().manual_seed(3)
    roll = lambda a, b: int(torch.randint(a, b + 1, (1,), generator=r))  # noqa: E731
    slot = lambda p: p if p < sinks else sinks + (p - sinks) % ring  # noqa: E731
    x, held, end, seen_end, both = rand(gen, 1, cap, D), {}, 0, 0, set()
    for i in range(600):
        kind = roll(0, 9)
        pos = end if kind < 7 else roll(0, end) if kind < 9 else 0
        n = roll(1, min(ring, 6))
        kv.write(0, pos, x[:, :n].contiguous(), x[:, :n].contiguous())
        held.update({slot(p): p for p in range(pos, pos + n)})
        end, seen_end = pos + n, max(seen_end, pos + n)
        rows = min(n, 5)
        if (end - rows >= sinks) or not sinks:
            assert attend_rc(kv, 0, rand(gen, 1, 1, D), end - 1, window=rows)[0] == 0
        for _ in range(4):
            total, window, keep = roll(1, seen_end), roll(1, 5), roll(0, sinks)
            want = set(range(max(0, total - window), total)) | set(range(min(keep, total)))
            rc = attend_rc(kv, 0, rand(gen, 1, 1, D), total - 1, window=window, sinks=keep)[0]
            ok = all(held.get(slot(p)) == p for p in want)
            both.add((rc == 0, ok))
            assert ok or rc == -1, (i, total, window, keep)
    assert (True, True) in both and (False, False) in both


def test_captured_writes_overwrite_nothing_before_they_run(gen):
    """A graph of the next positions' writes and attention, captured ahead: earlier positions stay open to eager calls."""
    D, window = 64, 10
    kv = cuda.KVCache.shaped(1, 2, D, 14, window=window)
    x, y, q = rand(gen, 2, 14, D), rand(gen, 2, 4, D), rand(gen, 1, 4, D)
    kv.write(0, 0, x, x)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    first = attend_rc(kv, 0, q, 9, window=window)[1]
    out = torch.empty_like(q)
    ws = torch.empty(cuda.attn_workspace_bytes(D), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        st = torch.cuda.current_stream().cuda_stream
        kv.write(0, 14, y, y, st)
        cuda.check(cuda.lib().mlxd_cuda_kv_attend(kv.kv, 0, q.data_ptr(), 256, 1, 17,
                                                  C.byref(cuda.attn_config(4, window=window)), out.data_ptr(), 256,
                                                  ws.data_ptr(), ws.numel(), st), "attend")
    rc, again, _ = attend_rc(kv, 0, q, 9, window=window)
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(first, again)
    g.replay()
    torch.cuda.synchronize()
    flat = cuda.KVCache.shaped(1, 2, D, 18)
    flat.write(0, 0, torch.cat((x, y), 1), torch.cat((x, y), 1))
    rc, want, _ = attend_rc(flat, 0, q, 17, window=window)
    torch.cuda.synchronize()
    assert rc == 0
    # the same keys in another order of slots: f32 sums of a few terms, each weight off by at most 2 * 2^-17
    bound = 2.0 ** -15 * x.double().abs().max() + 2.0 ** -7 * want.double().abs()
    assert bool(((out.double() - want.double()).abs() <= bound).all())


# ------------------------------------------------------------------ launches that gave up

def test_a_launch_that_gave_up_is_reported_to_its_own_caller(gen):
    """The words are set here as a launch would set them: no input makes a wait run out."""
    L = cuda.lib()
    a, b = (cache(gen, 2, 64, 300, 300) for _ in range(2))
    ga, gb = (Group(gen, 2, 64, 100, 100, 2, 8, layers=1, layer=0) for _ in range(2))
    q, lens, cfg = rand(gen, 40, 4, 64), torch.ones(2, dtype=torch.int32, device="cuda"), cuda.attn_config(4)
    for t in (ga, gb):
        t.fill([1, 1])
    calls = [lambda: a.attend(q, 200, cfg), lambda: b.attend(q, 200, cfg), lambda: ga.attend(q[:2], lens, cfg),
             lambda: gb.attend(q[:2], lens, cfg)]
    words = [L.mlxd_cuda_kv_gave_up(a.kv.kv), L.mlxd_cuda_kv_gave_up(b.kv.kv), L.mlxd_cuda_kv_group_gave_up(ga.g.g),
             L.mlxd_cuda_kv_group_gave_up(gb.g.g)]
    assert len({C.addressof(w.contents) for w in words}) == 4
    want = [f() for f in calls]
    torch.cuda.synchronize()
    for i, w in enumerate(words):
        assert [x[0] for x in words] == [0] * 4
        w[0] = 1
        for j, f in enumerate(calls):
            if j == i:
                with pytest.raises(cuda.CudaError, match="gave up"):
                    f()
            assert torch.equal(f(), want[j])
    assert not L.mlxd_cuda_kv_gave_up(None) and not L.mlxd_cuda_kv_group_gave_up(None)


def test_gave_up_words_come_and_go_with_their_caches(gen):
    """More caches than one page of words serves, some destroyed with their word set: new ones begin with zero."""
    L = cuda.lib()
    for _ in range(3):
        kvs = [cuda.KVCache.shaped(1, 1, 8, 4) for _ in range(150)]
        words = [L.mlxd_cuda_kv_gave_up(kv.kv) for kv in kvs]
        assert len({C.addressof(w.contents) for w in words}) == 150 and all(w[0] == 0 for w in words)
        for w in words[::2]:
            w[0] = 1
        for kv in kvs:
            kv.close()


@pytest.mark.parametrize("n", [1, 40])
def test_attend_scale_range(gen, n):
    """Scales whose product with log2 e leaves f32 are refused; the ends of the range weigh equal scores equally."""
    c = cache(gen, 2, 64, 200, 200)
    q = torch.zeros(n, 8, 64, device="cuda", dtype=torch.bfloat16)
    want = c.attend(q, 100, cuda.attn_config(8))
    for scale in (1e-30, 1.0, 1e30):
        assert torch.equal(c.attend(q, 100, cuda.attn_config(8, scale=scale)), want)
    for scale in (1e-31, 1e-45, 1.1e30, 3e38, math.inf, -1.0, math.nan):
        with pytest.raises(cuda.CudaError, match="bad attention parameters"):
            c.attend(q, 100, cuda.attn_config(8, scale=scale))


# ------------------------------------------------------------------ rotary positions against the model's own

@pytest.mark.parametrize("llama3", [None, (8.0, 1.0, 4.0, 64), (32.0, 1.0, 4.0, 8192)])
def test_rope_turns_as_the_models_cache_rows(llama3):
    """The same token at every position: the first layer's cached key at position 0 is the projection itself (cosine 1,
    sine 0), the others are its rotations by the model's table. That one's angles are products in f32 (off by 2^-23 of
    themselves), its cosines f32, the rows bf16; the op's angles are exact."""
    n, D, hkv, theta = 300, 64, 2, 1e4
    cfg = cuda.synth_config(hidden=256, layers=1, n_heads=4, n_kv_heads=hkv, head_dim=D, inter=256, vocab=256,
                            family=cuda.LLAMA, theta=theta, llama3=llama3, max_pos=512)
    m = cuda.Model(cfg, cuda.synth_host_tensors(cfg, seed=4, std=0.1))
    kv = m.new_kv(n)
    m.forward(kv, [7] * 200)
    for _ in range(200, n):                      # the decode step's rows, too
        m.forward(kv, [7])
    rows = kv.read(0)                            # [hkv][n][D]
    r = cuda.rope_config(theta, D)
    if llama3:
        r = cuda.rope_config(theta, D, scaling=cuda.ROPE_LLAMA3, factor=llama3[0], lo=llama3[1], hi=llama3[2],
                             orig_max=llama3[3])
    x = np.repeat(rows[None, :, 0], n, 0)        # [n][hkv][D]
    got = bf16_to_f32(cuda.rope(x, r, 0)).astype(np.float64)
    want = bf16_to_f32(rows).astype(np.float64).transpose(1, 0, 2)
    a = np.abs(bf16_to_f32(x).astype(np.float64))
    pair = np.concatenate((a[..., :D // 2] + a[..., D // 2:],) * 2, -1)
    p = np.arange(n)[:, None, None]
    bound = pair * (p * 2.0 ** -22 + 2.0 ** -20) + (np.abs(got) + np.abs(want)) * 2.0 ** -8
    assert np.all(np.abs(got - want) <= bound)
    assert np.abs(want).max() > 0.01 and not np.array_equal(want[1:], want[:-1])


# ------------------------------------------------------------------ two callers at once

def test_attend_on_two_streams_at_once(gen):
    """Calls of every form on two streams, a workspace each, over one cache and a group of its prefix: the bits of the
    same calls alone."""
    c = cache(gen, 4, 128, 3000, 3000)
    t = cuda.KVGroup(c.kv, 2500, 6, 40)
    x = rand(gen, 6, 4, 40, 128)
    for i in range(6):
        t.write(0, i, 0, x[i].contiguous(), (-x[i]).contiguous())
    lens = torch.tensor([1, 40, 7, 0, 33, 12], dtype=torch.int32, device="cuda")
    L, cfg, wide = cuda.lib(), cuda.attn_config(16), cuda.attn_config(32)
    calls = [(rand(gen, n, h, 128, scale=1.5), pos, a) for n, pos, h, a in ((1, 2999, 16, cfg), (700, 2000, 32, wide),
                                                                         (40, 2900, 16, cfg), (1, 50, 16, cfg))]
    qg = rand(gen, 6, 16, 128)

    def passes(ws, st):
        outs = []
        for q, pos, a in calls:
            o = torch.empty_like(q)
            cuda.check(L.mlxd_cuda_kv_attend(c.kv.kv, 0, q.data_ptr(), q.stride(0), q.shape[0], pos, C.byref(a),
                                             o.data_ptr(), o.stride(0), ws.data_ptr(), ws.numel(), st), "attend")
            outs.append(o)
        o = torch.empty_like(qg)
        cuda.check(L.mlxd_cuda_kv_group_attend(t.g, 0, qg.data_ptr(), qg.stride(0), lens.data_ptr(), C.byref(cfg),
                                               o.data_ptr(), o.stride(0), ws.data_ptr(), ws.numel(), st), "group")
        return outs + [o]

    ws = [torch.empty(cuda.attn_workspace_bytes(128), dtype=torch.uint8, device="cuda") for _ in range(2)]
    want = passes(ws[0], torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for w, s in zip(ws, streams):
            with torch.cuda.stream(s):
                got.append(passes(w, s.cuda_stream))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
