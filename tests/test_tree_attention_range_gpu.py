"""Tree attention where a row's probabilities, or its V scales, span a wide range; the
formula evaluated in 64 bits."""
import math

import pytest

from _util import torch_dtype

pytestmark = pytest.mark.gpu

# rows per cached head: every block size of both kernels
ROWS = [(1, 1), (3, 1), (12, 1), (20, 1), (50, 1), (30, 4)]


@pytest.mark.parametrize("T,G", ROWS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("far", [100.0, 150.0, 400.0])
def test_zero_value_row_with_all_the_weight(ltm, far, d, T, G):
    """int8: a key whose value row is zero (scale 0) scores `far` (in log2) above all others:
    the output is at most 2^-far of the values, nothing beside it in bf16's normal numbers
    at that, and never a NaN."""
    import torch
    n = 700
    g = torch.Generator().manual_seed(1)
    v = torch.randint(-127, 128, (1, 1, n + T, d), generator=g, dtype=torch.int8).cuda()
    vs = torch.full((1, 1, n + T), 0.01, device="cuda")
    k = torch.zeros((1, 1, n + T, d), dtype=torch.int8, device="cuda")
    ks = torch.ones((1, 1, n + T), device="cuda")
    k[:, :, 300] = 1
    ks[:, :, 300] = far * math.log(2.0) * math.sqrt(d) / (d * 4.0)
    v[:, :, 300] = 0
    vs[:, :, 300] = 0
    q = torch.full((1, T, G, d), 4.0, device="cuda").bfloat16()
    lens = torch.full((1,), n, dtype=torch.int32, device="cuda")
    got = ltm.tree_attention(q, k, v, lens, None, ks, vs).double()
    assert torch.isfinite(got).all()
    assert float(got.abs().max()) <= (n + T) * 1.27 * 2.0 ** (1 - far) + 2.0 ** -126


@pytest.mark.parametrize("T,G", ROWS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("others", [0.0, 0.01, 1e30])
@pytest.mark.parametrize("below", [0.0, 130.0])
def test_nan_scale_reaches_every_token_that_sees_it(ltm, below, others, d, T, G):
    """int8: a value row with the scale NaN (a row that held a NaN) whose key is seen gives
    NaN, whatever its weight and the others' scales; a drafted one only to its descendants."""
    import torch
    n = 300
    v = torch.full((1, 1, n + T, d), 100, dtype=torch.int8, device="cuda")
    vs = torch.full((1, 1, n + T), others, device="cuda")
    if others == 0:
        v.zero_()
    k = torch.zeros((1, 1, n + T, d), dtype=torch.int8, device="cuda")
    ks = torch.ones((1, 1, n + T), device="cuda")
    q = torch.full((1, T, G, d), 4.0, device="cuda").bfloat16()
    lens = torch.full((1,), n, dtype=torch.int32, device="cuda")
    for at, seen in ((150, range(T)), (n + T - 1, [T - 1])):
        v2, vs2, k2, ks2 = v.clone(), vs.clone(), k.clone(), ks.clone()
        v2[:, :, at] = 0
        vs2[:, :, at] = float("nan")
        k2[:, :, at] = -1
        ks2[:, :, at] = below * math.log(2.0) * math.sqrt(d) / (d * 4.0)
        got = ltm.tree_attention(q, k2, v2, lens, None, ks2, vs2)
        for t in range(T):
            bad = torch.isnan(got[0, t])
            assert bad.all() if t in seen else not bad.any(), (at, t)


@pytest.mark.parametrize("T,G", ROWS)
@pytest.mark.parametrize("cache", ["f16", "bf16", "int8"])
@pytest.mark.parametrize("d", [64, 128])
def test_many_small_probabilities(ltm, d, cache, T, G):
    """16 keys of value 0 (one for each warp) take nearly all of the weight; n others,
    2^-26 of one each, hold values of 64: o = 64 n 2^-26 / (16 + n 2^-26), about 2^-8.  More
    heads than SMs, so that a CTA goes through whole heads.

    Bound: the weights are rounded to 16 bits; those of f16 products are held relative to at
    least 2^7 for the largest, so that half a step below the normal numbers, 2^-25, is
    2^-32 of the largest, n 2^-32 64 / 16 in all; bf16 2^-8 relative.  The scores are those of
    exactly representable q and k, |score| <= 26 in units of log2: 26 2^-21 relative for the
    fp32 factor and the exponential.  The output rounds by half a step."""
    import torch
    n, heads, out_t = 65536, 160, "f16" if cache == "f16" else "bf16"
    td = torch_dtype(out_t)
    # q . k sl2 = -26 for every key but the 16 (all zeros)
    qv = 8.0
    kv = -26.0 * math.log(2.0) * math.sqrt(d) / (d * qv)
    q = torch.full((1, T, heads * G, d), qv, dtype=td, device="cuda")
    P = n + T
    if cache == "int8":
        k = torch.full((1, heads, P, d), -127, dtype=torch.int8, device="cuda")
        ks = torch.full((1, heads, P), -kv / 127, device="cuda")
        v = torch.full((1, heads, P, d), 127, dtype=torch.int8, device="cuda")
        vs = torch.full((1, heads, P), 64 / 127, device="cuda")
    else:
        k = torch.full((1, heads, P, d), kv, dtype=td, device="cuda")
        v = torch.full((1, heads, P, d), 64.0, dtype=td, device="cuda")
        ks = vs = None
    k[:, :, :256:16] = 0
    v[:, :, :256:16] = 0
    kk, vv = k[0, 0].double(), v[0, 0].double()
    if cache == "int8":
        kk, vv = kk * ks[0, 0].double()[:, None], vv * vs[0, 0].double()[:, None]
    lens = torch.full((1,), n, dtype=torch.int32, device="cuda")
    root = torch.full((1, T), -1, dtype=torch.int32, device="cuda")  # every token sees itself only
    got = ltm.tree_attention(q, k, v, lens, root, ks, vs).double()
    s = (kk[:n + 1] @ q[0, 0, 0].double()) / math.sqrt(d)
    want = float((torch.softmax(s, 0) @ vv[:n + 1])[0])
    assert 2.0 ** -9 < want < 2.0 ** -7
    u = 2.0 ** -8 if cache == "bf16" else 2.0 ** -11
    bound = want * (u + 26 * 2.0 ** -21) + (0 if cache == "bf16" else n * 2.0 ** -30)
    bound += want * (2.0 ** -11 if out_t == "f16" else 2.0 ** -8)
    assert torch.isfinite(got).all()
    assert float((got - want).abs().max()) <= bound, (float(got.min()), float(got.max()), want)
