"""KV cache writes, reads and reorders (ltm_kv_cache_append / _read / _reorder)
on the GPU.  Codes and scales are compared bit for bit with an IEEE evaluation of
the quantizer's formula in numpy, moved rows bit for bit with numpy indexing."""
import numpy as np
import pytest

from _util import torch_dtype

pytestmark = pytest.mark.gpu


def quant_rows(x):
    """fp32 [..., d] -> (int8 codes, fp32 scales): the documented formula."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        bad = ~np.isfinite(x).all(-1)
        a = np.where(np.isfinite(x), np.abs(x), 0).max(-1).astype(np.float32)
        s = (a / np.float32(127)).astype(np.float32)
        t = (x / np.where(s == 0, np.float32(1), s)[..., None]).astype(np.float32)
        lo = np.floor(np.abs(t))
        r = np.sign(t) * (lo + (np.abs(t) - lo >= np.float32(0.5)))
        q = np.where(bad[..., None] | (s == 0)[..., None], 0, np.clip(np.nan_to_num(r), -127, 127))
    return q.astype(np.int8), np.where(bad, np.float32(np.nan), s).astype(np.float32)


def fused_kv(B, T, h, d, dt, seed):
    """K and V as slices of fused projection rows [B, T, 3, h, d]."""
    import torch
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((B, T, 3, h, d), generator=g).to(torch_dtype(dt)).cuda()
    return qkv[:, :, 1], qkv[:, :, 2]


CASES = [(1, 1, 1, 64, 9), (3, 1, 5, 128, 40), (2, 7, 12, 64, 33), (2, 33, 2, 128, 70),
         (1, 130, 3, 64, 131), (5, 16, 1, 128, 19)]


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("B,T,h,d,P", CASES)
def test_append_int8_bit_exact(ltm, dt, B, T, h, d, P):
    import torch
    k, v = fused_kv(B, T, h, d, dt, B * 1000 + T)
    k[0, 0, 0] = 0                     # a zero row: scale 0, codes 0
    v[0, 0, 0, ::2] = 0.5              # ties of the rounding: 0.5 of amax 127
    v[0, 0, 0, 0] = 127
    lens = [(P - T) * b // max(1, B - 1) for b in range(B)]
    num = [T - (b % 3 if b % 3 < T else 0) for b in range(B)]
    kc = torch.full((B, h, P, d), 77, dtype=torch.int8, device="cuda")
    vc = torch.full_like(kc, 78)
    ks = torch.full((B, h, P), 5.0, device="cuda")
    vs = torch.full_like(ks, 6.0)
    i32 = dict(dtype=torch.int32, device="cuda")
    ltm.kv_cache_append(k, v, kc, vc, torch.tensor(lens, **i32), ks, vs, torch.tensor(num, **i32))
    for x, c, s, fc, fs in ((k, kc, ks, 77, 5.0), (v, vc, vs, 78, 6.0)):
        q, sc = quant_rows(x.float().cpu().numpy().transpose(0, 2, 1, 3))
        wc = np.full((B, h, P, d), fc, np.int8)
        ws = np.full((B, h, P), fs, np.float32)
        for b in range(B):
            wc[b, :, lens[b]:lens[b] + num[b]] = q[b, :, :num[b]]
            ws[b, :, lens[b]:lens[b] + num[b]] = sc[b, :, :num[b]]
        assert np.array_equal(c.cpu().numpy(), wc)
        assert np.array_equal(s.cpu().numpy(), ws)
    assert ltm.device_error() == 0


@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_append_rounds_like_the_division(ltm, dt):
    """Values at and next to the ties of every row's scale: rows whose largest values
    take every bf16 mantissa (and some of every other type's), values that are
    (n + 1/2) * amax / 127 moved by a few units in the last place, either sign, over many
    magnitudes."""
    import torch
    T, h, d = 128, 16, 128
    g = torch.Generator().manual_seed(1)
    top = (1 + torch.arange(T) / 128)[:, None] * (2.0 ** (8 * torch.arange(h) - 100).double())[None]
    if dt != "bf16":
        top = top * (1 + torch.rand((T, h), generator=g, dtype=torch.float64) / 200)
    if dt == "f16":
        top = top * 2.0 ** 100 / 2.0 ** (8 * torch.arange(h) - torch.arange(h) % 13 + 3).double()
    n = torch.randint(0, 127, (T, h, d), generator=g).double() + 0.5
    x = (n / 127 * top.to(torch_dtype(dt)).double()[..., None]).to(torch_dtype(dt))
    bits = torch.int32 if dt == "f32" else torch.int16
    step = torch.randint(-2, 3, (T, h, d), generator=g)
    x = (x.view(bits) + step.to(bits)).view(torch_dtype(dt))
    x[:, :, 5] = top.to(torch_dtype(dt))
    x = torch.minimum(x, x[:, :, 5:6]) * (1 - 2 * torch.randint(0, 2, (T, h, d), generator=g)).to(x.dtype)
    x = x[None].cuda()
    kc = torch.zeros((1, h, T, d), dtype=torch.int8, device="cuda")
    vc, ks = kc.clone(), torch.zeros((1, h, T), device="cuda")
    vs = ks.clone()
    ltm.kv_cache_append(x, -x, kc, vc, torch.zeros(1, dtype=torch.int32, device="cuda"), ks, vs)
    for y, c, s in ((x, kc, ks), (-x, vc, vs)):
        q, sc = quant_rows(y.float().cpu().numpy().transpose(0, 2, 1, 3))
        assert np.array_equal(s.cpu().numpy(), sc)
        assert np.array_equal(c.cpu().numpy(), q)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
def test_append_same_type_copies(ltm, dt, d):
    import torch
    B, T, h, P = 3, 19, 4, 50
    k, v = fused_kv(B, T, h, d, dt, 3)
    lens = [0, 31, 7]
    kc = torch.zeros((B, h, P, d), dtype=torch_dtype(dt), device="cuda")
    vc = torch.zeros_like(kc)
    ltm.kv_cache_append(k, v, kc, vc, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    for b in range(B):
        for x, c in ((k, kc), (v, vc)):
            assert torch.equal(c[b, :, lens[b]:lens[b] + T], x[b].transpose(0, 1))
            assert not c[b, :, :lens[b]].any() and not c[b, :, lens[b] + T:].any()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_append_extreme_rows(ltm, dt):
    """Tiny rows (scales in the subnormals), the largest finite values, and rows
    with an infinity or a NaN (scale NaN, codes 0; their reads are NaN)."""
    import torch
    td = torch_dtype(dt)
    B, T, h, d, P = 1, 9, 1, 64, 9
    rng = np.random.default_rng(4)
    x = rng.standard_normal((B, T, h, d)).astype(np.float32)
    tiny = float(torch.finfo(td).smallest_normal)
    x[0, 1] *= 1e-38
    x[0, 2] = np.where(np.arange(d) % 2, tiny, -tiny)
    x[0, 3] = np.arange(d) * 2.0 ** (-24 if dt == "f16" else -133 if dt == "bf16" else -149)
    x[0, 4] = np.where(np.arange(d) % 3, 1, -1) * float(torch.finfo(td).max)
    x[0, 5, 0, 3] = np.inf
    x[0, 6, 0, 5] = np.nan
    x[0, 7, 0, 9] = -np.inf
    x[0, 8] *= 1e-30
    with np.errstate(over="ignore"):
        k = torch.from_numpy(x).to(td).cuda()
    kc = torch.zeros((B, h, P, d), dtype=torch.int8, device="cuda")
    vc = torch.zeros_like(kc)
    ks, vs = torch.zeros((B, h, P), device="cuda"), torch.zeros((B, h, P), device="cuda")
    ltm.kv_cache_append(k, k, kc, vc, torch.zeros(1, dtype=torch.int32, device="cuda"), ks, vs)
    q, s = quant_rows(k.float().cpu().numpy().transpose(0, 2, 1, 3))
    for c, sc in ((kc, ks), (vc, vs)):
        assert np.array_equal(c.cpu().numpy(), q)
        assert np.array_equal(sc.cpu().numpy(), s, equal_nan=True)
    y = ltm.kv_cache_read(kc, ks, P).cpu().numpy()
    # reads are the fp32 product (amax = the largest fp32 value: its scale rounds up, so that
    # 127 * s passes the largest value and the formula itself gives an infinity)
    with np.errstate(over="ignore"):
        want = q.astype(np.float32) * s[..., None]
    same = np.array_equal(y, want, equal_nan=True)
    assert same and np.isnan(y[0, 0, 5:8]).all()


def test_append_skips_bad_lengths(ltm):
    import torch
    B, T, h, d, P = 5, 4, 2, 64, 10
    k, v = fused_kv(B, T, h, d, "bf16", 8)
    kc = torch.zeros((B, h, P, d), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    i32 = dict(dtype=torch.int32, device="cuda")
    # beyond the cache, negative, the last that fits, a count above T, a count of 0
    ltm.kv_cache_append(k, v, kc, vc, torch.tensor([7, -1, 6, 0, 10], **i32), None, None,
                        torch.tensor([4, 4, 4, 5, 0], **i32))
    torch.cuda.synchronize()
    assert ltm.device_error() == 5
    assert not kc[[0, 1, 3, 4]].any() and not vc[[0, 1, 3, 4]].any()
    assert torch.equal(kc[2, :, 6:], k[2].transpose(0, 1)) and not kc[2, :, :6].any()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,h,P,d,n", [(1, 1, 3, 64, 3), (2, 3, 41, 128, 17), (3, 12, 100, 64, 100),
                                       (1, 2, 300, 128, 257)])
def test_read_int8(ltm, dt, B, h, P, d, n):
    import torch
    rng = np.random.default_rng(n)
    q = rng.integers(-127, 128, (B, h, P, d)).astype(np.int8)
    s = rng.random((B, h, P)).astype(np.float32)
    first = [(b * 5) % 7 - 1 for b in range(B)]       # -1: its first row is outside
    lens = [P - 3 * b for b in range(B)]
    i32 = dict(dtype=torch.int32, device="cuda")
    out = torch.full((B, h, n, d), 9.0, dtype=torch_dtype(dt), device="cuda")
    got = ltm.kv_cache_read(torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda(), n,
                            first=torch.tensor(first, **i32), cache_lens=torch.tensor(lens, **i32),
                            dtype=torch_dtype(dt), out=out)
    assert got is out
    full = torch.from_numpy(q.astype(np.float32) * s[..., None]).to(torch_dtype(dt))
    for b in range(B):
        for i in range(n):
            p = first[b] + i
            want = full[b, :, p] if 0 <= p < lens[b] else torch.zeros_like(full[b, :, 0])
            assert torch.equal(out[b, :, i].cpu(), want), (b, i)


def test_read_16bit_and_defaults(ltm):
    import torch
    c = torch.randn((2, 3, 21, 64), device="cuda").bfloat16()
    assert torch.equal(ltm.kv_cache_read(c, None, 21), c)
    assert torch.equal(ltm.kv_cache_read(c, None, 30)[:, :, :21], c)
    assert not ltm.kv_cache_read(c, None, 30)[:, :, 21:].any()
    assert ltm.kv_cache_read(c, None, 0).shape == (2, 3, 0, 64)


# ------------------------------------------------------------------- reorder --
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 13, 32])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_reorder_any_map(ltm, W, kind):
    """Random maps (copies and drops), a cycle and the identity; K, V and the
    scales of an int8 cache in one call; ragged ranges; bytes outside untouched."""
    import torch
    B, h, P, d = 3, 2, 37, 64
    rng = np.random.default_rng(W)
    beams = rng.integers(0, W, (B, W)).astype(np.int32)
    beams[1] = np.roll(np.arange(W), 1)
    beams[2] = np.arange(W)
    beams[2, 0] = W - 1
    caches = []
    for _ in range(2):
        if kind == "int8":
            caches.append(torch.from_numpy(rng.integers(-127, 128, (B * W, h, P, d)).astype(np.int8)))
            caches.append(torch.from_numpy(rng.random((B * W, h, P)).astype(np.float32)))
        else:
            caches.append(torch.from_numpy(rng.standard_normal((B * W, h, P, d)).astype(np.float32))
                          .bfloat16())
    lens, first = [P, 20, 5], [0, 3, 5]
    want = []
    for t in caches:
        y = t.clone()
        for b in range(B):
            for w in range(W):
                y[b * W + w, :, first[b]:lens[b]] = t[b * W + beams[b, w], :, first[b]:lens[b]]
        want.append(y)
    dev = [t.cuda() for t in caches]
    i32 = dict(dtype=torch.int32, device="cuda")
    ltm.kv_cache_reorder(dev, torch.from_numpy(beams).cuda(), torch.tensor(lens, **i32),
                         torch.tensor(first, **i32))
    for got, y in zip(dev, want):
        assert torch.equal(got.cpu(), y)
    assert ltm.device_error() == 0


def test_reorder_many_caches_and_whole_range(ltm):
    """More caches than one launch takes; no lengths: all positions."""
    import torch
    caches = [torch.randn((4, 1, 3, 64), device="cuda").half() for _ in range(70)]
    want = [t[[1, 0, 3, 3]].clone() for t in caches]
    ltm.kv_cache_reorder(caches, torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("beams,lens,first", [([[0, 2]], [3], [0]), ([[-1, 0]], [3], [0]),
                                              ([[1, 0]], [9], [0]), ([[1, 0]], [2], [3]),
                                              ([[1, 0]], [3], [-1])])
def test_reorder_refuses_bad_requests_on_the_device(ltm, beams, lens, first):
    """The bad request keeps its caches, the other one is moved."""
    import torch
    c = torch.randn((4, 2, 8, 64), device="cuda").half()
    want = c.clone()
    want[2:, :, :4] = c[[3, 2], :, :4]
    i32 = dict(dtype=torch.int32, device="cuda")
    ltm.kv_cache_reorder([c], torch.tensor(beams + [[1, 0]], **i32), torch.tensor(lens + [4], **i32),
                         torch.tensor(first + [0], **i32))
    torch.cuda.synchronize()
    assert ltm.device_error() == 6
    assert torch.equal(c, want)
