"""Argument checks of the single ops for callers that drive layers themselves
(rotary positions, token scores, caches of a given shape, attention): every
refusal that needs no device, through the C ABI."""
import ctypes as C

import numpy as np
import pytest
import torch

from mlxd_b200 import cuda

X = np.zeros(4096, np.float32)


def refused(rc, word):
    assert rc == -1
    msg = cuda.lib().mlxd_cuda_last_error().decode()
    assert word in msg, msg


def rope(cfg=None, dtype=cuda.F32, n=1, heads=1, D=8, xs=(8, 8), pos=0, ys=(8, 8)):
    cfg = cfg or cuda.rope_config(1e4, 8)
    return cuda.lib().mlxd_cuda_rope(cuda.ptr(X), dtype, n, heads, D, *xs, C.byref(cfg), None, pos, cuda.ptr(X),
                                     *ys, None)


@pytest.mark.parametrize("kw", [dict(dtype=cuda.U32), dict(n=-1), dict(heads=0), dict(heads=65536), dict(D=1),
                                dict(D=264), dict(cfg=cuda.rope_config(1e4, 7)), dict(cfg=cuda.rope_config(1e4, 10)),
                                dict(cfg=cuda.rope_config(1e4, -2))])
def test_rope_refuses_bad_shapes(kw):
    refused(rope(**kw), "rope: bad arguments")


@pytest.mark.parametrize("kw", [dict(ys=(8, 4), heads=2), dict(ys=(4, 8), n=2), dict(xs=(-8, 8)), dict(ys=(-8, 8)),
                                dict(ys=(8, 8), n=2, heads=2), dict(ys=(20, 12), n=2, heads=3),
                                dict(ys=(8, 2 ** 62), heads=3)])
def test_rope_refuses_strides(kw):
    refused(rope(**kw), "rows of y overlap")


@pytest.mark.parametrize("cfg", [cuda.rope_config(0.0, 8), cuda.rope_config(1.0, 8), cuda.rope_config(float("nan"), 8),
                                 cuda.rope_config(1e4, 8, scaling=4), cuda.rope_config(1e4, 8, scaling=-1),
                                 cuda.rope_config(1e4, 8, scaling=cuda.ROPE_LINEAR, factor=0.5),
                                 cuda.rope_config(1e4, 8, scaling=cuda.ROPE_LLAMA3, factor=8, lo=4, hi=4),
                                 cuda.rope_config(1e4, 8, scaling=cuda.ROPE_LLAMA3, factor=8, lo=0, hi=4),
                                 cuda.rope_config(1e4, 8, scaling=cuda.ROPE_YARN, factor=8, lo=1, hi=32, orig_max=0),
                                 cuda.rope_config(1e4, 8, scaling=cuda.ROPE_YARN, factor=float("inf"), lo=1, hi=32),
                                 cuda.rope_config(1e4, 8, scaling=cuda.ROPE_YARN, factor=8, lo=1, hi=32,
                                                  magnitude=-1)])
def test_rope_refuses_parameters(cfg):
    refused(rope(cfg=cfg), "rope: invalid base or scaling")


def test_rope_refuses_position_overflow_and_null_config():
    refused(rope(pos=2 ** 31 - 2, n=2), "overflows")
    refused(cuda.lib().mlxd_cuda_rope(cuda.ptr(X), cuda.F32, 1, 1, 8, 8, 8, None, None, 0, cuda.ptr(X), 8, 8, None),
            "bad arguments")


def test_empty_calls_do_nothing():
    assert rope(n=0) == 0
    assert scores(rows=0) == 0


def scores(dtype=cuda.F32, rows=1, V=64, stride=64, targets=X, top=4, lp=X):
    p = lambda a: cuda.ptr(a) if a is not None else None  # noqa: E731
    return cuda.lib().mlxd_cuda_token_scores(cuda.ptr(X), dtype, rows, V, stride, p(targets), top, p(lp), None,
                                             cuda.ptr(X), cuda.ptr(X), None)


@pytest.mark.parametrize("kw", [dict(dtype=cuda.I32), dict(rows=-1), dict(V=0), dict(stride=-1), dict(top=-1),
                                dict(top=33), dict(V=3, top=4)])
def test_scores_refuse_bad_arguments(kw):
    refused(scores(**kw), "token_scores: bad arguments")


def test_scores_refuse_logprobs_without_targets():
    refused(scores(targets=None), "without targets")


@pytest.mark.parametrize("args,word", [((0, 1, 64, 8, 0, 0), "bad arguments"), ((1, 0, 64, 8, 0, 0), "bad arguments"),
                                       ((1, 1, 60, 8, 0, 0), "bad arguments"), ((1, 1, 264, 8, 0, 0), "bad arguments"),
                                       ((1, 1, 64, 0, 0, 0), "bad arguments"), ((1, 1, 64, 8, -1, 0), "bad arguments"),
                                       ((1, 1, 64, 8, 0, 2), "sinks without a window"),
                                       ((1, 1, 64, 8, 7, 2), "smaller than 2 sinks and the window 7")])
def test_shaped_cache_refuses(args, word):
    h = C.c_void_p(7)
    refused(cuda.lib().mlxd_cuda_kv_create_shape(C.byref(h), *args), word)
    assert h.value == 7      # out-parameters are written only on success


def test_attention_refuses_null_handles():
    cfg = cuda.attn_config(8)
    L, p = cuda.lib(), cuda.ptr(X)
    refused(L.mlxd_cuda_kv_attend(None, 0, p, 64, 1, 0, C.byref(cfg), p, 64, p, 0, None), "kv_attend: bad arguments")
    refused(L.mlxd_cuda_kv_group_attend(None, 0, p, 64, p, C.byref(cfg), p, 64, p, 0, None), "bad arguments")
    refused(L.mlxd_cuda_kv_group_append(None, 0, p, 64, p, 64, p, None), "bad arguments")
    refused(L.mlxd_cuda_kv_group_write(None, 0, 0, 0, 1, p, p, None), "bad arguments")
    h = C.c_void_p(7)
    refused(L.mlxd_cuda_kv_group_create(C.byref(h), None, 0, 1, 8), "bad arguments")
    assert h.value == 7
    L.mlxd_cuda_kv_group_destroy(None)


def test_workspace_size_is_known_without_a_device():
    assert cuda.attn_workspace_bytes(128) > 0
    assert cuda.attn_workspace_bytes(128) >= cuda.attn_workspace_bytes(64)
    assert cuda.attn_workspace_bytes(0) == 0


def test_host_wrappers_refuse_lengths_that_do_not_match():
    x = np.zeros((3, 2, 8), np.float32)
    for pos in (np.arange(2), np.arange(4), np.zeros((3, 1))):
        with pytest.raises(ValueError, match="positions for 3 tokens"):
            cuda.rope(x, cuda.rope_config(1e4, 8), pos)
    for targets in ([1, 2], [1, 2, 3, 4], 1):
        with pytest.raises(ValueError, match="targets for 3 rows"):
            cuda.token_scores(np.zeros((3, 16), np.float32), targets)


@pytest.mark.parametrize("k,v", [((2, 5, 16), (2, 4, 16)), ((2, 5, 16), (1, 5, 16)), ((3, 5, 16), (3, 5, 16)),
                                 ((2, 5, 8), (2, 5, 8)), ((10, 16), (10, 16))])
def test_cache_rows_refuse_shapes(k, v):
    with pytest.raises(ValueError, match="cache rows"):
        cuda.row_count(torch.zeros(k, dtype=torch.bfloat16), torch.zeros(v, dtype=torch.bfloat16), (2, 16))


def test_cache_rows_refuse_strides_and_types():
    a = torch.zeros(2, 5, 16, dtype=torch.bfloat16)
    assert cuda.row_count(a, a, (2, 16)) == 5
    for b in (a.transpose(0, 1).contiguous().transpose(0, 1), a[:, ::2], a.float()):
        with pytest.raises(ValueError, match="cache rows"):
            cuda.row_count(b, b, (2, 16))


@pytest.mark.parametrize("V", [2 ** 31 - 1, 2 ** 31 - 256])
def test_scores_refuse_rows_whose_steps_pass_the_int_range(V):
    refused(scores(V=V, stride=V), "token_scores: bad arguments")


def test_cache_rows_refuse_other_16_bit_floats():
    a = torch.zeros(2, 5, 16, dtype=torch.bfloat16)
    for b in (a, a.view(torch.int16), a.view(torch.uint16)):
        assert cuda.row_count(b, b, (2, 16)) == 5
    for k, v in ((a.half(), a), (a, a.half())):
        with pytest.raises(ValueError, match="cache rows"):
            cuda.row_count(k, v, (2, 16))


def test_cache_rows_refuse_host_memory():
    """Before the library is called with the address."""
    kv = cuda.KVCache.__new__(cuda.KVCache)
    kv.model, kv.kv, kv.shape = None, None, (2, 16)
    g = cuda.KVGroup.__new__(cuda.KVGroup)
    g.g, g.prefix = None, kv
    a = torch.zeros(2, 5, 16, dtype=torch.bfloat16)
    for f in (lambda: kv.write(0, 0, a, a), lambda: g.write(0, 0, 0, a, a)):
        with pytest.raises(ValueError, match="device memory"):
            f()
