"""Beam selection's branches by size: many rows of 16-bit logits (16384 of them a CTA), more
continuations to merge than shared memory holds, the merge of equal totals one by one; and
rows whose totals lie so far out that 64 bits tell few logits apart."""
import numpy as np
import pytest

from _util import torch_dtype
from test_beam_gpu import check

pytestmark = pytest.mark.gpu


def rows(B, W, V, dt, seed, off=1):
    """Logits whose rows start off a 16-byte boundary, `off` elements on."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    big = torch.empty((B, W, V + off + 3), dtype=torch_dtype(dt), device="cuda")
    big.copy_(4 * torch.randn(big.shape, generator=g, device="cuda"))
    scores = -20 * torch.rand((B, W), generator=g, device="cuda")
    done = torch.rand((B, W), generator=g, device="cuda") < 0.2
    return big[:, :, off:off + V], scores, done


# rows x chunks of 8192 must pass four times the SMs for 16384 logits a CTA
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("V", [8193, 16385, 32001])
@pytest.mark.parametrize("off,K", [(0, 16), (1, 16), (5, 16), (1, 17), (3, 64)])
def test_many_rows(ltm, dt, V, off, K):
    import torch
    W = 8
    B = 4 * torch.cuda.get_device_properties(0).multi_processor_count // (W * ((V + 8191) // 8192)) + 1
    x, scores, done = rows(B, W, V, dt, V + off, off)
    check(ltm, x, scores, K)
    check(ltm, x, scores, K, done, V - 1)
    x[0] = 1.5                      # equal logits, equal beams
    scores[0] = -3.0
    x[1, :, ::3] = float("nan")
    x[2, :, V // 3:] = float("-inf")
    x[3, 0, V - 1] = float("inf")
    x[3, 5, 0] = float("inf")
    x[4] = x[4].sort(-1).values
    x[5] = x[5].sort(-1, descending=True).values
    x[6] = torch.finfo(x.dtype).min
    x[6, 2, V - 2] = 0
    x[7] = x[7].round()
    check(ltm, x, scores, K)
    check(ltm, x, scores, K - 1, done, 0)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_more_lists_than_shared_memory_holds(ltm, dt):
    B, W, V, K = 2, 32, 40000, 64  # 32 x 5 x 64 = 10240 entries
    x, scores, done = rows(B, W, V, dt, 3)
    check(ltm, x, scores, K)
    check(ltm, x, scores, K, done, 7)


@pytest.mark.parametrize("K", [17, 64])
@pytest.mark.parametrize("W,V", [(32, 40000), (32, 8000), (12, 8192)])
def test_equal_totals_merged_one_by_one(ltm, W, V, K):
    import torch
    x, scores, _ = rows(2, W, V, "f16", 4)
    x[0] = 0.25
    scores[0] = -2.0
    out = check(ltm, x, scores, K)
    assert (out[1][0] == 0).all() and torch.equal(out[2][0].cpu(), torch.arange(K, dtype=torch.int32))
    scores[:] = -2.0  # and with a beam that is ahead of the rest, and one behind
    x[0, 3, 100] = 0.5
    x[0, 5, :] = 0.125
    check(ltm, x, scores, K)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [700, 20000])
@pytest.mark.parametrize("K", [4, 33])
def test_totals_that_64_bits_cannot_tell_apart(ltm, dt, V, K):
    """Scores of fp32's lowest value (beams that do not exist yet, written so) and logits of
    +inf: most totals of such a row are equal in 64 bits, and go by the lowest token."""
    import torch
    W = 4
    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn((6, W, V), generator=g)).to(torch_dtype(dt)).cuda()
    scores = torch.zeros((6, W), device="cuda")
    lowest = torch.finfo(torch.float32).min
    scores[:, 1:] = lowest
    x[0, 0, 2:] = float("-inf")          # the one beam has two tokens left
    x[1, 0] = float("-inf")              # or none
    x[2, 0, 1:] = float("-inf")
    x[2, 1, V // 2:] = torch.finfo(x.dtype).min
    x[3, :, V // 2] = float("inf")
    x[4, 1:, V - 1] = float("inf")
    scores[5] = torch.tensor([lowest, -1e30, -1e25, lowest])
    check_inf(ltm, x, scores, K)
    x = x[:, :1].contiguous()
    x[:, :, V - 2] = float("inf")
    check_inf(ltm, x, torch.zeros((6, 1), device="cuda"), K)


@pytest.mark.parametrize("dt", ["f32", "f16"])
@pytest.mark.parametrize("low", [-1e9, -3.4028234663852886e38])
def test_far_scores_beside_finished_beams(ltm, dt, low):
    """Finished beams, whose end token is masked among their logits, between beams of far
    scores with few tokens left."""
    import torch
    B, W, V, K, end = 24, 7, 8193, 14, 3212
    g = torch.Generator().manual_seed(6)
    x = (10 * torch.randn((B, W, V), generator=g)).to(torch_dtype(dt)).cuda()
    x[(torch.rand(x.shape, generator=g) < 0.999).cuda()] = float("-inf")
    x[:, :, end] = float("-inf")
    scores = -20 * torch.rand((B, W), generator=g).cuda()
    scores[:, 1:] = low
    done = (torch.rand((B, W), generator=g) < 0.3).cuda()
    check(ltm, x, scores, K, done, end)
    check(ltm, x, scores, K)


def check_inf(ltm, x, scores, K):
    """+inf counts as the type's largest value."""
    import torch
    want = check(ltm, x.clamp(max=torch.finfo(x.dtype).max), scores, K)
    got = ltm.beam_select(x, scores, K)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
