"""Tree attention where a row's probabilities, or its V scales, span a wide range; the
formula evaluated in 64 bits."""
import math

import pytest

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
