"""Workloads of the operators for callers that drive decoder layers themselves:
rotary positions, attention over a KV cache (sliding window with sink positions),
attention for a batch that shares a prefix, and token scores.

Each case has a plain form (elementary torch operations) and the call that a user
makes of libmlxd_cuda (taken where `own` is true); exact() restates the operators
in 64 bits from their definitions.
"""
import math

import torch

own = False

ROPE_DEFAULT, ROPE_LINEAR, ROPE_LLAMA3, ROPE_YARN = 0, 1, 2, 3
SCALINGS = {"default": ROPE_DEFAULT, "linear": ROPE_LINEAR, "llama3": ROPE_LLAMA3, "yarn": ROPE_YARN}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one decode step's q and k heads of a 32/8-head model, in the fused projection's row
        dict(name="rope 1 token", op="rope", n=1, heads=40, D=128, dims=128, inter=False, scaling="default",
             theta=1e6, dtype="bf16", pos=2191, batch=False, extra=1024),
        # a batch of decode steps far into a long context: interleaved pairs on half of each head, YaRN, f32
        dict(name="rope yarn batch 77", op="rope", n=77, heads=20, D=128, dims=64, inter=True, scaling="yarn",
             theta=1e4, dtype="f32", pos=120000, batch=True, extra=0),
        # a whole prompt's q and k heads of a 64/8-head model with llama3 frequencies
        dict(name="rope llama3 prompt 8192", op="rope", n=8192, heads=72, D=128, dims=128, inter=False,
             scaling="llama3", theta=5e5, dtype="bf16", pos=0, batch=False, extra=1024),
        # the logprobs of one sampled token with its five alternatives
        dict(name="scores 1 row", op="scores", rows=1, V=151936, top=5, dtype="bf16", pad=0),
        # a short odd batch over another vocabulary, f32 rows with a padded stride
        dict(name="scores 7 rows f32", op="scores", rows=7, V=32768, top=20, dtype="f32", pad=3),
        # scoring a 512-token chunk of a prompt, twenty alternatives
        dict(name="scores 512 rows", op="scores", rows=512, V=151936, top=20, dtype="bf16", pad=0),
        # a decode step at the benchmark's mean context
        dict(name="attend 1 token at 2192", op="attend", n=1, pos=2191, hq=32, hkv=8, D=128, cap=2561, window=0,
             sinks=0),
        # a decode step over a long cache
        dict(name="attend 1 token at 32768", op="attend", n=1, pos=32767, hq=32, hkv=8, D=128, cap=32768, window=0,
             sinks=0),
        # a prefill chunk over a wrapped ring: window 4096, four sink positions, 4607 ring slots
        dict(name="attend window chunk 512", op="attend", n=512, pos=7680, hq=32, hkv=8, D=128, cap=4611,
             window=4096, sinks=4),
        # the second half of an 8192-token prompt
        dict(name="attend chunk 4096 at 4096", op="attend", n=4096, pos=4096, hq=32, hkv=8, D=128, cap=8192,
             window=0, sinks=0),
        # eight samples of one prompt (16/8 heads)
        dict(name="shared 8 x 2048", op="shared", seqs=8, prefix=2048, tail=64, hq=16, hkv=8, D=128, window=0,
             sinks=0),
        # sixty-four samples of one long prompt, ragged tails
        dict(name="shared 64 x 8192", op="shared", seqs=64, prefix=8192, tail=512, hq=32, hkv=8, D=128, window=0,
             sinks=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "scores", "attend", "attend", "shared"])
    if op == "rope":
        D = rng.choice([16, 64, 80, 96, 128, 128])
        scaling = rng.choice(list(SCALINGS))
        return dict(op=op, n=_log(rng, 1, 8192), heads=rng.randint(1, 72), D=D,
                    dims=rng.choice([D, D, D // 2, D // 4]), inter=rng.random() < 0.4, scaling=scaling,
                    theta=rng.choice([1e4, 5e5, 1e6]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                    pos=_log(rng, 1, 200000) - 1, batch=rng.random() < 0.3, extra=rng.choice([0, 8, 1024, 3]))
    if op == "scores":
        return dict(op=op, rows=_log(rng, 1, 512), V=_log(rng, 500, 151936), top=rng.randint(0, 32),
                    dtype=rng.choice(["bf16", "bf16", "f32"]), pad=rng.choice([0, 0, 1, 8]))
    hkv, rep = rng.choice([(1, 8), (2, 4), (4, 7), (8, 1), (8, 2), (8, 4), (4, 8), (8, 4)])
    D = rng.choice([64, 80, 128, 128])
    if op == "shared":
        window = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
        return dict(op=op, seqs=_log(rng, 1, 64), prefix=_log(rng, 1, 8192), tail=_log(rng, 1, 512), hq=hkv * rep,
                    hkv=hkv, D=D, window=window, sinks=rng.choice([0, 4]) if window else 0)
    n = _log(rng, 1, 4096) if rng.random() < 0.6 else 1
    if rng.random() < 0.5:
        window, sinks = _log(rng, 16, 4096), rng.choice([0, 1, 4, 16])
        n = min(n, 1024)
        return dict(op=op, n=n, pos=_log(rng, 1, 20000) - 1, hq=hkv * rep, hkv=hkv, D=D,
                    cap=sinks + window + n - 1 + rng.randint(0, 300), window=window, sinks=sinks)
    pos = _log(rng, 1, 32768 if n == 1 else 4096) - 1
    return dict(op=op, n=n, pos=pos, hq=hkv * rep, hkv=hkv, D=D, cap=pos + n + rng.randint(0, 300), window=0, sinks=0)


# ------------------------------------------------------------------ shapes

def _slot_positions(cap, sinks, total, device):
    """Position held by each cache slot once positions [0, total) are written (-1: none). Position p lies in slot p
    below `sinks`, above in the ring of the other slots."""
    s = torch.arange(cap, device=device)
    ring = cap - sinks
    i = s - sinks
    last = total - 1 - sinks - i                    # >= 0 where position sinks + i is written
    p = torch.where(s < sinks, s, sinks + i + torch.div(last, ring, rounding_mode="floor") * ring)
    return torch.where(torch.where(s < sinks, s < total, last >= 0), p, torch.full_like(p, -1))


def _visible_counts(case):
    """(pairs of query and key, keys that any query sees) of an attend case."""
    n, pos, w, s = case["n"], case["pos"], case["window"], case["sinks"]
    if not w:
        return n * pos + n * (n + 1) // 2, pos + n
    near = [min(w, q + 1) for q in range(pos, pos + n)]
    far = [max(0, min(s, q + 1 - c)) for q, c in zip(range(pos, pos + n), near)]
    lo = max(0, pos - w + 1)
    return sum(near) + sum(far), pos + n - lo + min(s, lo)


def _tails(case, seed):
    g = torch.Generator().manual_seed(seed * 7 + 3)
    return torch.randint(1, case["tail"] + 1, (case["seqs"],), generator=g, dtype=torch.int32)


def work(case):
    op = case["op"]
    if op == "rope":
        e = 2 if case["dtype"] == "bf16" else 4
        els = case["n"] * case["heads"] * case["D"]
        return {"bytes": 2 * els * e + 4 * case["n"] * case["batch"],
                "flops": 3 * case["n"] * case["heads"] * case["dims"]}
    if op == "scores":
        e = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["rows"] * (case["V"] * e + 12 + 8 * case["top"]), "flops": 5 * case["rows"] * case["V"]}
    hq, hkv, D = case["hq"], case["hkv"], case["D"]
    if op == "attend":
        pairs, keys = _visible_counts(case)
        return {"bytes": 4 * case["n"] * hq * D + 4 * keys * hkv * D, "flops": 4 * pairs * hq * D}
    seqs, w = case["seqs"], case["window"]
    tail = (case["tail"] + 1) / 2                   # mean tail length
    tail_seen = min(tail, w) if w else tail
    pre_seen = min(case["prefix"], max(0, w - tail) + case["sinks"]) if w else case["prefix"]
    return {"bytes": 4 * seqs * hq * D + 4 * hkv * D * (pre_seen + seqs * tail_seen) + 4 * seqs,
            "flops": 4 * seqs * hq * D * (pre_seen + tail_seen)}


# ------------------------------------------------------------------ inputs

def _rand(g, *shape, dtype=torch.bfloat16, scale=1.0):
    x = torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32)
    return x.mul_(scale).to(dtype)


def _logits(case, g):
    """Rows like a decoder's: a broad bulk, a few likely tokens, and on every third row a vocabulary mask."""
    rows, V, dt = case["rows"], case["V"], DTYPES[case["dtype"]]
    x = torch.randn(rows, V + case["pad"], device="cuda", generator=g).mul_(2.5)
    hot = torch.randint(0, V, (rows, 12), device="cuda", generator=g)
    x.scatter_add_(1, hot, torch.rand(rows, 12, device="cuda", generator=g) * 14)
    blocked = torch.rand(V, device="cuda", generator=g) < 0.5
    x[::3, :V] = torch.where(blocked, torch.full_like(x[::3, :V], -math.inf), x[::3, :V])
    some = torch.randint(0, V, (rows, 1), device="cuda", generator=g)
    targets = torch.where(torch.rand(rows, 1, device="cuda", generator=g) < 0.5, hot[:, :1], some)
    return x.to(dt)[:, :V], targets[:, 0].to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    st = {"case": case}
    if own:
        from mlxd_b200 import cuda
        st["cuda"], st["lib"] = cuda, cuda.lib()
    if op == "rope":
        n, heads, D = case["n"], case["heads"], case["D"]
        row = heads * D + case["extra"]             # the heads lead a wider row (a fused projection)
        st["x"] = _rand(g, n, row, dtype=DTYPES[case["dtype"]])[:, :heads * D].unflatten(1, (heads, D))
        if case["batch"]:                           # each row at a position of its own
            st["pos"] = torch.randint(0, case["pos"] + 1, (n,), device="cuda", generator=g).to(torch.int32)
        if own:
            st["cfg"] = cuda.rope_config(case["theta"], case["dims"], interleaved=case["inter"],
                                         scaling=SCALINGS[case["scaling"]], **_scaling_args(case))
        return st
    if op == "scores":
        st["logits"], st["targets"] = _logits(case, g)
        return st
    hq, hkv, D = case["hq"], case["hkv"], case["D"]
    if op == "attend":
        n, pos, cap = case["n"], case["pos"], case["cap"]
        st["q"] = _rand(g, n, hq, D, scale=1.5)
        st["k"], st["v"] = _rand(g, hkv, cap, D), _rand(g, hkv, cap, D)
        if own:
            kv = cuda.KVCache.shaped(1, hkv, D, cap, window=case["window"], sinks=case["sinks"])
            at = _slot_positions(cap, case["sinks"], pos + n, "cuda")
            order = torch.argsort(at)[int((at < 0).sum()):]      # written slots by position
            ps = at[order].tolist()
            cut = next((i for i in range(1, len(ps)) if ps[i] != ps[i - 1] + 1), len(ps))
            for a, b in ((0, cut), (cut, len(ps))):              # the sinks, then the ring's positions
                if b > a:
                    kv.write(0, ps[a], st["k"][:, order[a:b]].contiguous(), st["v"][:, order[a:b]].contiguous())
            st["kv"] = kv
    else:
        seqs, prefix = case["seqs"], case["prefix"]
        st["q"] = _rand(g, seqs, hq, D, scale=1.5)
        st["k"], st["v"] = _rand(g, hkv, prefix, D), _rand(g, hkv, prefix, D)
        st["lens"] = _tails(case, seed).cuda()
        st["tk"], st["tv"] = _rand(g, seqs, hkv, case["tail"], D), _rand(g, seqs, hkv, case["tail"], D)
        if own:
            kv = cuda.KVCache.shaped(1, hkv, D, prefix)
            kv.write(0, 0, st["k"], st["v"])
            st["group"] = cuda.KVGroup(kv, prefix, seqs, case["tail"])
            for i, m in enumerate(st["lens"].tolist()):
                st["group"].write(0, i, 0, st["tk"][i, :, :m].contiguous(), st["tv"][i, :, :m].contiguous())
    if own:
        st["cfg"] = cuda.attn_config(hq, window=case["window"], sinks=case["sinks"])
        st["ws"] = torch.empty(cuda.attn_workspace_bytes(D), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
    return st


def _scaling_args(case):
    return {"default": {}, "linear": dict(factor=4.0),
            "llama3": dict(factor=8.0, lo=1.0, hi=4.0, orig_max=8192),
            "yarn": dict(factor=16.0, lo=1.0, hi=32.0, orig_max=8192)}[case["scaling"]]


# ------------------------------------------------------------------ the pass

def run(st):
    op = st["case"]["op"]
    if own:
        return {"rope": _own_rope, "scores": _own_scores, "attend": _own_attend, "shared": _own_shared}[op](st)
    return {"rope": _plain_rope, "scores": _plain_scores, "attend": _plain_attend, "shared": _plain_shared}[op](st)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_rope(st):
    c, x, cuda = st["case"], st["x"], st["cuda"]
    n, heads, D = x.shape
    y = torch.empty(n, heads, D, dtype=x.dtype, device=x.device)
    pos = st["pos"].data_ptr() if c["batch"] else None
    cuda.check(st["lib"].mlxd_cuda_rope(x.data_ptr(), cuda.BF16 if c["dtype"] == "bf16" else cuda.F32, n, heads, D,
                                        x.stride(0), x.stride(1), st["cfg"], pos, c["pos"], y.data_ptr(),
                                        y.stride(0), y.stride(1), _stream()), "rope")
    return y


def _own_scores(st):
    c, x, cuda = st["case"], st["logits"], st["cuda"]
    rows, top = c["rows"], c["top"]
    lp = torch.empty(rows, dtype=torch.float32, device=x.device)
    ent = torch.empty(rows, dtype=torch.float32, device=x.device)
    ids = torch.empty(rows, top, dtype=torch.int32, device=x.device)
    tlp = torch.empty(rows, top, dtype=torch.float32, device=x.device)
    cuda.check(st["lib"].mlxd_cuda_token_scores(x.data_ptr(), cuda.BF16 if c["dtype"] == "bf16" else cuda.F32, rows,
                                                c["V"], x.stride(0), st["targets"].data_ptr(), top, lp.data_ptr(),
                                                ent.data_ptr(), ids.data_ptr(), tlp.data_ptr(), _stream()),
               "token_scores")
    return {"logprob": lp, "entropy": ent, "ids": ids, "top": tlp}


def _own_attend(st):
    c, q, ws = st["case"], st["q"], st["ws"]
    out = torch.empty_like(q)
    st["cuda"].check(st["lib"].mlxd_cuda_kv_attend(st["kv"].kv, 0, q.data_ptr(), q.stride(0), c["n"], c["pos"],
                                                   st["cfg"], out.data_ptr(), out.stride(0), ws.data_ptr(),
                                                   ws.numel(), _stream()), "kv_attend")
    return out


def _own_shared(st):
    q, ws = st["q"], st["ws"]
    out = torch.empty_like(q)
    st["cuda"].check(st["lib"].mlxd_cuda_kv_group_attend(st["group"].g, 0, q.data_ptr(), q.stride(0),
                                                         st["lens"].data_ptr(), st["cfg"], out.data_ptr(),
                                                         out.stride(0), ws.data_ptr(), ws.numel(), _stream()),
                     "kv_group_attend")
    return out


def _inv_freq(c, device):
    """Inverse frequencies in 64 bits and the magnitude of the rotated features."""
    d, a = c["dims"], _scaling_args(c)
    i = torch.arange(0, d, 2, dtype=torch.float64, device=device)
    inv = c["theta"] ** (-i / d)
    if c["scaling"] == "linear":
        return inv / a["factor"], 1.0
    if c["scaling"] == "llama3":
        wl = 2 * math.pi / inv
        smooth = ((a["orig_max"] / wl - a["lo"]) / (a["hi"] - a["lo"])).clamp(0, 1)
        return inv * ((1 - smooth) / a["factor"] + smooth), 1.0
    if c["scaling"] == "yarn":
        turns = [a["hi"], a["lo"]]                  # the pair that turns so often over orig_max positions
        lo, hi = (d * math.log(a["orig_max"] / (t * 2 * math.pi)) / (2 * math.log(c["theta"])) for t in turns)
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), d - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv * (ramp / a["factor"] + 1 - ramp), 0.1 * math.log(a["factor"]) + 1
    return inv, 1.0


def _plain_rope(st):
    c, x = st["case"], st["x"]
    d = c["dims"]
    inv, mag = _inv_freq(c, x.device)
    pos = st["pos"] if c["batch"] else torch.arange(c["pos"], c["pos"] + c["n"], device=x.device)
    angle = pos.double()[:, None] * inv
    co, si = ((f(angle) * mag).float()[:, None, :] for f in (torch.cos, torch.sin))
    r = x[..., :d].float()
    a, b = (r[..., 0::2], r[..., 1::2]) if c["inter"] else (r[..., :d // 2], r[..., d // 2:])
    u, v = a * co - b * si, a * si + b * co
    r = torch.stack((u, v), -1).flatten(-2) if c["inter"] else torch.cat((u, v), -1)
    return torch.cat((r.to(x.dtype), x[..., d:]), -1)


def _plain_scores(st):
    c, x = st["case"], st["logits"].float()
    m = x.amax(1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    s = e.sum(1, keepdim=True, dtype=torch.float64)
    log_s = torch.log(s)
    weighted = torch.where(e > 0, e * z, torch.zeros_like(z)).sum(1, keepdim=True, dtype=torch.float64)
    t = st["targets"].long()[:, None]
    lp = (x.gather(1, t) - m).double() - log_s
    val, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top = (val[:, :c["top"]] - m).double() - log_s
    return {"logprob": lp[:, 0].float(), "entropy": (log_s - weighted / s)[:, 0].float(),
            "ids": ids[:, :c["top"]].to(torch.int32), "top": top.float()}


def _softmax_rows(s, mask):
    s = torch.where(mask, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    return e, e.sum(-1, keepdim=True)


def _seen(qpos, kpos, window, sinks):
    near = (qpos - kpos < window) | (kpos < sinks) if window else torch.ones_like(qpos - kpos, dtype=torch.bool)
    return (kpos >= 0) & (kpos <= qpos) & near


def _plain_attend(st):
    c, q = st["case"], st["q"]
    n, hq, D = q.shape
    hkv = c["hkv"]
    kpos = _slot_positions(c["cap"], c["sinks"], c["pos"] + n, q.device)
    qpos = torch.arange(c["pos"], c["pos"] + n, device=q.device)
    mask = _seen(qpos[:, None], kpos[None, :], c["window"], c["sinks"])          # [n][cap]
    qg = q.float().unflatten(1, (hkv, -1)).permute(1, 2, 0, 3).flatten(1, 2)      # [hkv][rep n][D]
    s = (qg @ st["k"].float().transpose(1, 2)) / math.sqrt(D)
    e, total = _softmax_rows(s.unflatten(1, (-1, n)), mask)
    out = e.flatten(1, 2) @ st["v"].float()
    out = out.unflatten(1, (-1, n)) / total.clamp(min=1e-38)
    return out.permute(2, 0, 1, 3).reshape(n, hq, D).to(q.dtype)


def _plain_shared(st):
    c, q, lens = st["case"], st["q"], st["lens"]
    n, hq, D = q.shape
    hkv, prefix, tail = c["hkv"], c["prefix"], c["tail"]
    qpos = prefix + lens[:, None].long() - 1
    kpos = torch.arange(prefix + tail, device=q.device)[None, :]
    mask = _seen(qpos, kpos, c["window"], c["sinks"])[:, None, None, :]           # [n][1][1][keys]
    qg = q.float().unflatten(1, (hkv, -1))                                        # [n][hkv][rep][D]
    s = torch.cat((qg @ st["k"].float().transpose(1, 2), qg @ st["tk"].float().transpose(2, 3)), -1) / math.sqrt(D)
    e, total = _softmax_rows(s, mask)
    out = (e[..., :prefix] @ st["v"].float() + e[..., prefix:] @ st["tv"].float()) / total.clamp(min=1e-38)
    return out.reshape(n, hq, D).to(q.dtype)


# ------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    with torch.no_grad():
        st = prepare(case, seed)
        return {"rope": _exact_rope, "scores": _exact_scores, "attend": _exact_attend,
                "shared": _exact_shared}[case["op"]](st)


def _exact_rope(st):
    """Every pair as a complex number, turned by its angle."""
    c, x = st["case"], st["x"].double()
    d, a = c["dims"], _scaling_args(c)
    inv, mag = [], 1.0
    for i in range(d // 2):
        f = math.exp(-2.0 * i / d * math.log(c["theta"]))
        if c["scaling"] == "linear":
            f = f / a["factor"]
        elif c["scaling"] == "llama3":
            turns = a["orig_max"] * f / (2 * math.pi)          # over the original context
            if turns < a["lo"]:
                f = f / a["factor"]
            elif turns <= a["hi"]:
                keep = (turns - a["lo"]) / (a["hi"] - a["lo"])
                f = keep * f + (1 - keep) * f / a["factor"]
        elif c["scaling"] == "yarn":
            mag = 1.0 + math.log(a["factor"]) / 10
            at = lambda t: math.log(a["orig_max"] / (2 * math.pi * t)) / math.log(c["theta"]) * d / 2  # noqa: E731
            lo, hi = max(math.floor(at(a["hi"])), 0), min(math.ceil(at(a["lo"])), d - 1)
            far = min(max((i - lo) / ((hi - lo) or 0.001), 0.0), 1.0)
            f = far * f / a["factor"] + (1 - far) * f
        inv.append(f)
    p = st["pos"].double() if c["batch"] else c["pos"] + torch.arange(c["n"], dtype=torch.float64, device=x.device)
    phase = torch.outer(p, torch.tensor(inv, dtype=torch.float64, device=x.device))
    turn = torch.polar(torch.full_like(phase, mag), phase)[:, None, :]
    y = x.clone()
    if c["inter"]:
        z = torch.complex(x[..., 0:d:2].contiguous(), x[..., 1:d:2].contiguous()) * turn
        y[..., 0:d:2], y[..., 1:d:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:d].contiguous()) * turn
        y[..., :d // 2], y[..., d // 2:d] = z.real, z.imag
    return y


def _exact_scores(st):
    c, x = st["case"], st["logits"]
    lp, ent, ids, top = [], [], [], []
    for r in range(c["rows"]):                      # a row at a time: log_softmax in 64 bits
        row = x[r].double()
        logp = row - torch.logsumexp(row, 0)
        lp.append(logp[st["targets"][r].long()])
        live = logp[logp > -math.inf]
        ent.append(-(torch.exp(live) * live).sum())
        order = torch.argsort(-row, stable=True)[:c["top"]]
        ids.append(order.to(torch.int32))
        top.append(logp[order])
    return {"logprob": torch.stack(lp), "entropy": torch.stack(ent), "ids": torch.stack(ids), "top": torch.stack(top)}


def _exact_attend(st):
    """Query by query block over the rows in position order."""
    c = st["case"]
    n, pos, cap, w, s, hkv = c["n"], c["pos"], c["cap"], c["window"], c["sinks"], c["hkv"]
    rep, D = c["hq"] // hkv, c["D"]
    total = pos + n
    first = max(0, pos - w + 1) if w else 0
    ps = sorted(set(range(min(s, total))) | set(range(first, total)))
    slot = torch.tensor([p if p < s else s + (p - s) % (cap - s) for p in ps], device="cuda")
    kp = torch.tensor(ps, device="cuda")
    out = torch.empty(n, c["hq"], D, dtype=torch.float64, device="cuda")
    for h in range(c["hq"]):
        k, v = st["k"][h // rep].double()[slot], st["v"][h // rep].double()[slot]
        for a in range(0, n, 1024):
            qp = torch.arange(pos + a, pos + min(a + 1024, n), device="cuda")[:, None]
            hide = kp > qp
            if w:
                hide = hide | ((kp <= qp - w) & (kp >= s))
            z = (st["q"][a:a + 1024, h].double() @ k.T) * D ** -0.5
            out[a:a + 1024, h] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ v
    return out


def _exact_shared(st):
    """Sequence by sequence, prefix and tail as one row of keys."""
    c = st["case"]
    hkv, rep, D = c["hkv"], c["hq"] // c["hkv"], c["D"]
    out = torch.empty(c["seqs"], c["hq"], D, dtype=torch.float64, device="cuda")
    for i, m in enumerate(st["lens"].tolist()):
        last = c["prefix"] + m - 1
        ps = [p for p in range(last + 1) if not c["window"] or last - p < c["window"] or p < c["sinks"]]
        at = torch.tensor(ps, device="cuda")
        k = torch.cat((st["k"], st["tk"][i, :, :m]), 1)[:, at].double()
        v = torch.cat((st["v"], st["tv"][i, :, :m]), 1)[:, at].double()
        q = st["q"][i].double().reshape(hkv, rep, D)
        z = torch.einsum("hrd,hkd->hrk", q, k) / D ** 0.5
        out[i] = torch.einsum("hrk,hkd->hrd", torch.softmax(z, -1), v).reshape(c["hq"], D)
    return out
