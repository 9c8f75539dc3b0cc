"""Refusals of the KV-cache and beam operators: argument errors come back from
the C ABI before any device call, and the Python layer checks shapes, types and
devices first (no GPU needed)."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import ltm_b200
    return ltm_b200.lib()


def _s(*v):
    return (C.c_int64 * len(v))(*v)


A = 1 << 20  # an aligned address that no refused call touches


def _append(lib, **kw):
    a = dict(k=A, ks=_s(256, 128, 64), v=A, vs=_s(256, 128, 64), dt=1, kc=A, vc=A, ksc=None,
             vsc=None, P=16, lens=A, num=None, B=1, T=2, h=2, d=64)
    a.update(kw)
    return lib.ltm_kv_cache_append(a["k"], a["ks"], a["v"], a["vs"], a["dt"], a["kc"], a["vc"],
                                   a["ksc"], a["vsc"], a["P"], a["lens"], a["num"], a["B"], a["T"],
                                   a["h"], a["d"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), 1), (dict(v=None), 1), (dict(kc=None), 1), (dict(lens=None), 1),
    (dict(ks=None), 1), (dict(ksc=A), 1), (dict(vsc=A), 1), (dict(k=A + 2), 1),
    (dict(kc=A + 8), 1), (dict(ks=_s(256, 129, 64)), 1), (dict(dt=3), 1), (dict(dt=0), 5),
    (dict(d=96), 5), (dict(P=0), 1), (dict(P=1 << 31), 1), (dict(h=0), 1), (dict(B=-1), 1),
    (dict(T=-1), 1), (dict(B=0), 0), (dict(T=0), 0)])
def test_append_refusals(lib, kw, status):
    assert _append(lib, **kw) == status
    assert bool(lib.ltm_last_error_string()) == (status != 0)


@pytest.mark.parametrize("kw,status", [
    (dict(cache=None), 1), (dict(out=None), 1), (dict(out=A + 4), 1), (dict(dt=4), 1),
    (dict(scale=None, dt=0), 5), (dict(d=32), 5), (dict(n=-1), 1), (dict(n=0), 0), (dict(B=0), 0)])
def test_read_refusals(lib, kw, status):
    a = dict(cache=A, scale=A, dt=1, P=16, B=1, h=2, d=64, n=4, out=A)
    a.update(kw)
    assert lib.ltm_kv_cache_read(a["cache"], a["scale"], a["dt"], a["P"], None, None, a["B"],
                                 a["h"], a["d"], a["n"], a["out"], None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(kc=None), 1), (dict(lens=None), 1), (dict(o=None), 1),
    (dict(ws=None), 1), (dict(ksc=A), 1), (dict(q=A + 2), 1), (dict(o=A + 4), 1),
    (dict(qs=_s(256, 132, 64)), 1), (dict(dt=0), 5), (dict(T=65), 5), (dict(d=80), 5),
    (dict(heads=3), 1), (dict(heads=256, kvh=2), 5), (dict(P=0), 1), (dict(T=0), 0),
    (dict(B=0), 0)])
def test_tree_refusals(lib, kw, status):
    a = dict(q=A, qs=_s(256, 128, 64), kc=A, vc=A, ksc=None, vsc=None, P=16, lens=A, o=A,
             os=_s(256, 128, 64), B=1, T=2, heads=2, kvh=2, d=64, dt=1, ws=A, n=1 << 20)
    a.update(kw)
    assert lib.ltm_tree_attention(a["q"], a["qs"], a["kc"], a["vc"], a["ksc"], a["vsc"], a["P"],
                                  a["lens"], None, None, a["o"], a["os"], a["B"], a["T"],
                                  a["heads"], a["kvh"], a["d"], a["dt"], a["ws"], a["n"],
                                  None) == status


def test_workspaces(lib):
    n = C.c_size_t()
    assert lib.ltm_tree_attention_workspace(4, 5, 8, 8, 64, C.byref(n)) == 0 and n.value > 0
    assert lib.ltm_tree_attention_workspace(4, 5, 8, 3, 64, C.byref(n)) == 1
    assert lib.ltm_tree_attention_workspace(4, 5, 8, 8, 64, None) == 1
    assert lib.ltm_beam_select_workspace(2, 4, 32000, 8, C.byref(n)) == 0 and n.value > 0
    assert lib.ltm_beam_select_workspace(2, 0, 32000, 8, C.byref(n)) == 1


@pytest.mark.parametrize("kw,status", [
    (dict(logits=None), 1), (dict(scores=None), 1), (dict(ws=None), 1), (dict(n=8), 1),
    (dict(ws=A + 4), 1), (dict(W=33), 5), (dict(K=65), 5), (dict(K=0), 1), (dict(V=0), 1),
    (dict(W=1, V=3, K=4), 1), (dict(dt=7), 1), (dict(done=A), 1), (dict(odone=A), 1),
    (dict(done=A, odone=A, end=-1), 1), (dict(done=A, odone=A, end=100), 1),
    (dict(logits=A + 1), 1), (dict(V=(1 << 24) + 1), 1), (dict(B=0), 0)])
def test_beam_refusals(lib, kw, status):
    a = dict(logits=A, dt=1, scores=A, done=None, end=0, B=1, W=2, V=100, K=2, odone=None, ws=A,
             n=1 << 20)
    a.update(kw)
    assert lib.ltm_beam_select(a["logits"], a["dt"], 200, 100, a["scores"], a["done"], a["end"],
                               a["B"], a["W"], a["V"], a["K"], A, A, A, a["odone"], a["ws"],
                               a["n"], None) == status


def _ptrs(*v):
    return (C.c_void_p * len(v))(*v)


@pytest.mark.parametrize("kw,status", [
    (dict(caches=None), 1), (dict(beams=None), 1), (dict(caches=_ptrs(A, None)), 1),
    (dict(caches=_ptrs(A, A)), 1), (dict(rows=_s(128, 6)), 1), (dict(rows=_s(0, 128)), 1),
    (dict(caches=_ptrs(A + 4, 2 * A)), 1), (dict(W=33), 5), (dict(W=0), 1), (dict(P=0), 1),
    (dict(n=0), 0), (dict(B=0), 0)])
def test_reorder_refusals(lib, kw, status):
    a = dict(caches=_ptrs(A, 2 * A), rows=_s(128, 4), n=2, beams=A, B=1, W=2, h=2, P=16)
    a.update(kw)
    assert lib.ltm_kv_cache_reorder(a["caches"], a["rows"], a["n"], a["beams"], None, None, a["B"],
                                    a["W"], a["h"], a["P"], None) == status


def test_python_layer_refuses_cpu_tensors():
    import ltm_b200 as ltm
    import torch
    x = torch.zeros((1, 1, 1, 64), dtype=torch.float16)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ltm.kv_cache_append(x, x, x, x, n)
    with pytest.raises(ValueError):
        ltm.kv_cache_read(x, None, 1)
    with pytest.raises(ValueError):
        ltm.tree_attention(x, x, x, n)
    with pytest.raises(ValueError):
        ltm.beam_select(torch.zeros((1, 1, 4)), torch.zeros((1, 1)))
    with pytest.raises(ValueError):
        ltm.kv_cache_reorder([x], torch.zeros((1, 1), dtype=torch.int32))
