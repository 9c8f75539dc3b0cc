"""Caches, inputs and outputs past 2^31 elements: what is written and read lies where 64-bit
index arithmetic puts it, and nothing beside it changes."""
import pytest
import torch

from test_beam_gpu import check

pytestmark = pytest.mark.gpu

H, P, D = 8, 800_001, 128  # 3 sequences: 2.46e9 elements


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def quantised(x):
    """Codes and scales of the formula (rows without ties here)."""
    s = x.float().abs().amax(-1)
    s = s / torch.full_like(s, 127.0)
    return torch.round(x.float() / s[..., None]).to(torch.int8), s


@pytest.mark.parametrize("cache", ["int8", "f16"])
def test_write_and_read(ltm, cache):
    B, T = 3, 37
    assert B * H * P * D > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(0)
    ct = torch.int8 if cache == "int8" else torch.float16
    kc, vc = (torch.zeros((B, H, P, D), dtype=ct, device="cuda") for _ in range(2))
    ks = vs = None
    if cache == "int8":
        ks, vs = (torch.zeros((B, H, P), device="cuda") for _ in range(2))
    k, v = (torch.randn((B, T, H, D), generator=g, device="cuda").half() for _ in range(2))
    lens = i32(0, P // 2, P - T)
    ltm.kv_cache_append(k, v, kc, vc, lens, ks, vs)
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        back = ltm.kv_cache_read(c, s, T, first=lens, dtype=torch.float16)
        for b, at in enumerate(lens.tolist()):
            rows = x[b].transpose(0, 1)
            if s is None:
                want = rows
                assert torch.equal(c[b, :, at:at + T], rows)
            else:
                q, sc = quantised(rows)
                far = (c[b, :, at:at + T].int() - q.int()).abs().max()
                assert far <= 1 and torch.equal(s[b, :, at:at + T], sc)  # torch rounds ties to even
                want = (c[b, :, at:at + T].float() * sc[..., None]).half()
            assert torch.equal(back[b], want)
            assert not c[b, :, :at].any() and not c[b, :, at + T:].any()
    assert ltm.device_error() == 0


def test_read_of_a_whole_cache(ltm):
    """The output past 2^31 elements, too."""
    g = torch.Generator(device="cuda").manual_seed(1)
    c = torch.randint(-127, 128, (3, H, P, D), generator=g, dtype=torch.int8, device="cuda")
    s = torch.rand((3, H, P), generator=g, device="cuda")
    got = ltm.kv_cache_read(c, s, P, dtype=torch.float16)
    for b in range(3):
        for h in range(H):
            assert torch.equal(got[b, h], (c[b, h].float() * s[b, h][:, None]).half())


def test_inputs_far_apart(ltm):
    """Token rows and logits whose batches lie 2^31 elements apart."""
    far = 2 ** 31 + 4096
    big = torch.zeros((far + 4096,), dtype=torch.float16, device="cuda")
    x = torch.as_strided(big, (2, 3, 2, D), (far, 2 * D, D, 1))
    x.copy_(torch.randn(x.shape, device="cuda").half())
    kc, vc = (torch.zeros((2, 2, 16, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ltm.kv_cache_append(x, x, kc, vc, i32(1, 13))
    for c in (kc, vc):
        assert torch.equal(c[0, :, 1:4], x[0].transpose(0, 1))
        assert torch.equal(c[1, :, 13:16], x[1].transpose(0, 1))
        assert not c[0, :, 4:].any() and not c[1, :, :13].any()
    o = torch.as_strided(big, x.shape, x.stride(), 3 * 2 * D)
    want = ltm.tree_attention(x, kc, vc, i32(1, 13))
    assert ltm.tree_attention(x, kc, vc, i32(1, 13), out=o) is o and torch.equal(o, want)
    logits = torch.as_strided(big, (2, 3, 1000), (far, 1001, 1))
    logits.copy_(torch.randn(logits.shape, device="cuda").half())
    scores = -torch.rand((2, 3), device="cuda")
    check(ltm, logits, scores, 5)


def test_reorder(ltm):
    """4 beams of 1 request; a cycle and a copy at the far end of the caches."""
    c = torch.zeros((4, 2, 3_000_000, D), dtype=torch.float16, device="cuda")
    q = torch.zeros((4, 2, 3_000_000, D), dtype=torch.int8, device="cuda")
    s = torch.zeros((4, 2, 3_000_000), device="cuda")
    assert c.numel() > 2 ** 31 and q.numel() > 2 ** 31
    lo, hi = 2_999_000, 2_999_991
    far = slice(lo, hi)
    for x in (c, q, s):
        n = x[:, :, far].numel()
        x[:, :, far] = torch.randint(1, 100, (n,), device="cuda").view(x[:, :, far].shape).to(x.dtype)
    beams = [2, 0, 1, 1]
    want = [torch.stack([x[w, :, far] for w in beams]) for x in (c, q, s)]
    ltm.kv_cache_reorder([c, q, s], i32(*beams).view(1, 4), i32(hi), first=i32(lo))
    for x, y in zip((c, q, s), want):
        assert torch.equal(x[:, :, far], y)
        assert not x[:, :, hi:].any() and not x[:, :, lo - 1000:lo].any()
    assert ltm.device_error() == 0


def test_read_of_a_very_long_sequence(ltm):
    """More positions than one launch takes (65535 blocks of 64)."""
    n = 65535 * 64 + 100
    c = torch.zeros((1, 1, n, D), dtype=torch.int8, device="cuda")
    c[0, 0, :, 0] = torch.arange(n, device="cuda") % 127
    c[0, 0, :, 1] = torch.arange(n, device="cuda") // 65536
    s = torch.ones((1, 1, n), device="cuda")
    got = ltm.kv_cache_read(c, s, n, first=i32(3), cache_lens=i32(n - 5))
    assert torch.equal(got[0, 0, :n - 8], c[0, 0, 3:n - 5].float())
    assert not got[0, 0, n - 8:].any()
