"""The Python layer of the KV-cache and beam operators refuses tensors that do not
fit together, before any launch (their memory stays as it was)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture
def t(ltm):
    """Tensors of one valid call of each operator."""
    import torch
    dev = dict(device="cuda")
    B, T, h, d, P, W, V = 2, 3, 2, 64, 16, 4, 100
    x = dict(k=torch.randn((B, T, h, d), **dev).half(), kc=torch.zeros((B, h, P, d), **dev).half(),
             q8=torch.zeros((B, h, P, d), dtype=torch.int8, **dev),
             s=torch.zeros((B, h, P), **dev), lens=torch.zeros(B, dtype=torch.int32, **dev),
             par=torch.full((B, T), -1, dtype=torch.int32, **dev),
             logits=torch.randn((B, W, V), **dev), scores=torch.zeros((B, W), **dev),
             done=torch.zeros((B, W), dtype=torch.bool, **dev),
             beams=torch.zeros((B, W), dtype=torch.int32, **dev),
             beamc=torch.zeros((B * W, h, P, d), **dev).half())
    x["vc"], x["v8"], x["s2"] = x["kc"].clone(), x["q8"].clone(), x["s"].clone()
    return x


def refused(ltm, f, status=1):
    with pytest.raises(ltm.LtmError) as e:
        f()
    assert e.value.status == status and str(e.value)


def test_append_refusals(ltm, t):
    import torch
    k, kc, vc, q8, v8, s, s2, n = (t[x] for x in ("k", "kc", "vc", "q8", "v8", "s", "s2", "lens"))
    f = ltm.kv_cache_append
    f(k, k, kc, vc, n)
    f(k, k, q8, v8, n, s, s2)
    for args in ((k[:1], k, kc, vc, n), (k, k.bfloat16(), kc, vc, n), (k[0], k[0], kc, vc, n),
                 (k, k, kc[:, :1], vc[:, :1], n), (k, k, kc.transpose(1, 2), vc, n),
                 (k, k, kc.bfloat16(), vc.bfloat16(), n), (k, k, kc, vc, n.long()),
                 (k, k, kc, vc, n[:1]), (k, k, q8, v8, n), (k, k, kc, vc, n, s, s2),
                 (k, k, q8, v8, n, s, None), (k, k, q8, v8, n, s.half(), s2),
                 (k, k, q8, v8, n, s[:, :, :8], s2), (k, k, q8, vc, n, s, None),
                 (k[..., ::2], k[..., ::2], kc, vc, n), (k[..., 1:33], k[..., 1:33], kc, vc, n),
                 (k, k, kc, vc, n, None, None, n.float())):
        refused(ltm, lambda: f(*args))
    refused(ltm, lambda: f(k[..., :32], k[..., :32], kc[..., :32].contiguous(),
                           vc[..., :32].contiguous(), n), 5)
    refused(ltm, lambda: f(k.float(), k.float(), kc.float(), vc.float(), n), 5)
    with pytest.raises((TypeError, ValueError)):
        f(k, k, kc, vc, [0, 0])
    with pytest.raises((TypeError, ValueError)):
        f(k, k, kc, vc, None)
    refused(ltm, lambda: f(k, k, kc, vc, n.cpu()))
    assert torch.cuda.current_device() == 0 and ltm.device_error() == 0


def test_read_and_tree_refusals(ltm, t):
    import torch
    k, kc, vc, q8, v8, s, s2, n = (t[x] for x in ("k", "kc", "vc", "q8", "v8", "s", "s2", "lens"))
    f = ltm.kv_cache_read
    for args, kw in (((q8, None, 3), {}), ((kc, s, 3), {}), ((q8, s, -1), {}),
                     ((kc, None, 3), dict(dtype=torch.float32)),
                     ((q8, s, 3), dict(dtype=torch.float64)),
                     ((q8, s, 3), dict(out=torch.empty((2, 2, 4, 64), device="cuda"))),
                     ((q8, s, 3), dict(first=n.long())), ((q8, s, 3), dict(cache_lens=n[:1]))):
        refused(ltm, lambda: f(*args, **kw))
    g = ltm.tree_attention
    assert g(k, kc, vc, n, t["par"]).shape == k.shape
    for args, kw in (((k, kc, vc, n, t["par"][:, :2]), {}), ((k, kc, vc, n, t["par"].long()), {}),
                     ((k.bfloat16(), kc, vc, n), {}), ((k[:1], kc, vc, n), {}),
                     ((k, q8, v8, n), {}), ((k, q8, v8, n), dict(k_scale=s)),
                     ((k[:, :, :1].expand(2, 3, 3, 64), kc, vc, n), {}),
                     ((k, kc, vc, n), dict(out=k.float())), ((k, kc, vc, n), dict(out=k[:1])),
                     ((k.transpose(2, 3), kc, vc, n), {})):
        refused(ltm, lambda: g(*args, **kw))
    refused(ltm, lambda: g(torch.zeros((2, 65, 2, 64), device="cuda").half(), kc, vc, n), 5)
    refused(ltm, lambda: g(k.float(), q8, v8, n, None, s, s2), 5)
    assert g(k[:, :0], kc, vc, n).shape == (2, 0, 2, 64)
    assert g(k[:0], kc[:0], vc[:0], n[:0]).shape == (0, 3, 2, 64)


def test_beam_and_reorder_refusals(ltm, t):
    import torch
    x, sc, dn = t["logits"], t["scores"], t["done"]
    f = ltm.beam_select
    assert f(x, sc)[0].shape == (2, 4)
    for args, kw in (((x, sc.double()), {}), ((x, sc[:, :2]), {}), ((x, sc.t()), {}),
                     ((x[0], sc), {}), ((x.transpose(1, 2), sc), {}), ((x, sc, 0), {}),
                     ((x, sc, 4), dict(done=dn)), ((x, sc, 4), dict(done=dn.int(), end_token=1)),
                     ((x, sc, 4), dict(done=dn, end_token=100)), ((x.double(), sc), {}),
                     ((x[:, :, :1], sc, 5), {})):
        refused(ltm, lambda: f(*args, **kw))
    refused(ltm, lambda: f(x, sc, 65), 5)
    assert f(x[:0], sc[:0])[1].shape == (0, 4)
    c, b = t["beamc"], t["beams"]
    g = ltm.kv_cache_reorder
    g([c], b)
    for args in (([c, c], b), ([c[:2]], b), ([c, c[:, :1].contiguous()], b), ([c], b.long()),
                 ([c], b[0]), ([c.transpose(0, 1)], b), ([c], b, t["lens"][:1]),
                 ([c, c[0, 0]], b)):
        refused(ltm, lambda: g(*args))
    g([], b)
    with pytest.raises((TypeError, ValueError)):
        g([c, None], b)
