"""Beam selection (ltm_beam_select) on the GPU against a plain evaluation in 64
bits.

Scores: the row's sum of exponentials is taken in fp32 (at most 40 additions in
a chain, 2^-24 each; the exponential's error is a few 2^-23 for the terms that count), so a
log-probability is off by less than 5e-6, plus half a step of the fp32 result.  The
selection must be that of the reference wherever neighbouring totals differ by more
than 1e-5; equal totals (equal logits of a row, equal beams) go by the flat index."""
import numpy as np
import pytest

from _util import torch_dtype

pytestmark = pytest.mark.gpu


def reference(logits, scores, done, end):
    """fp64 totals [B, W * V]."""
    x = logits.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    m = x.max(-1, keepdims=True)
    m0 = np.where(np.isfinite(m), m, 0)
    with np.errstate(divide="ignore", invalid="ignore"):
        lse = np.log(np.exp(x - m0).sum(-1, keepdims=True))
        s = np.where(np.isnan(scores), -np.inf, scores).astype(np.float64)
        t = s[..., None] + ((x - m0) - lse)
    t = np.where(np.isneginf(x) | np.isneginf(s)[..., None], -np.inf, t)
    if done is not None:
        only = np.full_like(t, -np.inf)
        only[..., end] = s
        t = np.where(done[..., None], only, t)
    return t.reshape(t.shape[0], -1)


def check(ltm, logits, scores, K, done=None, end=-1):
    """Runs the kernel on device tensors and compares with the reference."""
    import torch
    B, W, V = logits.shape
    out = ltm.beam_select(logits, scores, K, done=done, end_token=end)
    s, beams, tokens = (t.cpu().numpy() for t in out[:3])
    d = None if done is None else done.cpu().numpy()
    t = reference(logits.float().cpu().numpy(), scores.cpu().numpy(), d, end)
    flat = beams.astype(np.int64) * V + tokens
    for b in range(B):
        order = np.argsort(-t[b], kind="stable")[:K + 1]
        want = t[b][order]
        assert len(set(flat[b])) == K, "a continuation twice"
        for k in range(K):
            if flat[b, k] != order[k]:  # only where the totals cannot be told apart
                assert abs(t[b][flat[b, k]] - want[k]) < 1e-5, (b, k)
                same_row = flat[b, k] // V == order[k] // V
                assert not same_row or t[b][flat[b, k]] != want[k], "a tie by the wrong index"
            if np.isneginf(want[k]):
                assert np.isneginf(s[b, k])
                assert flat[b, k] == order[k]
            else:
                assert abs(s[b, k] - want[k]) <= 5e-6 + 2.0 ** -24 * abs(want[k]), (b, k)
    if done is not None:
        fin = out[3].cpu().numpy()
        assert np.array_equal(fin, np.take_along_axis(d, beams, 1) | (tokens == end))
    assert ltm.device_error() == 0
    return out


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,W,V,K", [(1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 7, 16), (1, 4, 1000, 4),
                                     (3, 5, 8192, 10), (2, 4, 8193, 8), (1, 2, 32000, 64),
                                     (2, 8, 50001, 16), (1, 32, 700, 32), (4, 1, 16385, 1)])
def test_matches_reference(ltm, dt, B, W, V, K):
    import torch
    g = torch.Generator().manual_seed(V + K)
    logits = (3 * torch.randn((B, W, V), generator=g)).to(torch_dtype(dt)).cuda()
    scores = (-10 * torch.rand((B, W), generator=g)).cuda()
    check(ltm, logits, scores, K)
    done = (torch.rand((B, W), generator=g) < 0.4).cuda()
    check(ltm, logits, scores, K, done, V // 2)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_first_step_and_dead_beams(ltm, dt):
    """Only beam 0 exists at first; then no beam at all."""
    import torch
    logits = torch.randn((2, 4, 5000), generator=torch.Generator().manual_seed(1))
    logits = logits.to(torch_dtype(dt)).cuda()
    scores = torch.full((2, 4), float("-inf"), device="cuda")
    scores[:, 0] = 0
    out = check(ltm, logits, scores, 8)
    assert not out[1].any()
    scores[1] = float("-inf")
    scores[0, 1] = float("nan")
    check(ltm, logits, scores, 8)
    done = torch.zeros((2, 4), dtype=torch.bool, device="cuda")
    done[1] = True
    check(ltm, logits, scores, 8, done, 3)


@pytest.mark.parametrize("V", [600, 20000])
@pytest.mark.parametrize("K", [1, 8, 33])
def test_ties_and_masks(ltm, V, K):
    """Equal logits everywhere, equal beams, all but a few masked with -inf or with the
    type's lowest value, a block masked, sorted rows, NaN, +inf."""
    import torch
    rng = np.random.default_rng(V + K)
    W = 3
    x = rng.standard_normal((10, W, V)).astype(np.float32)
    x[0] = 1.5
    x[1] = x[1, :1]
    x[2] = -np.inf
    x[2, :, rng.choice(V, 5, replace=False)] = 2.0
    x[3, :, V // 3:] = -np.inf
    x[4] = np.sort(x[4], -1)
    x[5] = np.sort(x[5], -1)[:, ::-1]
    x[6, :, ::3] = np.nan
    x[7, 0, 7] = np.inf
    x[7, 1, [3, 9]] = np.inf
    x[8] = np.finfo(np.float32).min
    x[8, 1, V - 1] = 0
    x[9] = np.round(x[9])
    x[9, :, ::2] = 0.0
    x[9, :, 1::2] = -0.0
    scores = np.zeros((10, W), np.float32)
    scores[4:] = -rng.random((6, W)).astype(np.float32)
    check(ltm, torch.from_numpy(x).cuda(), torch.from_numpy(scores).cuda(), K)


def test_row_with_no_token_left(ltm):
    import torch
    x = torch.zeros((1, 2, 100), device="cuda")
    x[0, 0] = float("-inf")
    out = check(ltm, x, torch.zeros((1, 2), device="cuda"), 5)
    assert (out[1] == 1).all()
    check(ltm, torch.full((1, 2, 100), float("-inf"), device="cuda"),
          torch.zeros((1, 2), device="cuda"), 5)


@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_strided_and_misaligned_rows(ltm, dt):
    """Rows that start at any element of a 16-byte unit; strides between them."""
    import torch
    g = torch.Generator().manual_seed(3)
    big = (2 * torch.randn((2, 3, 9007), generator=g)).to(torch_dtype(dt)).cuda()
    scores = -torch.rand((2, 3), generator=g).cuda()
    for off in range(0, 9):
        check(ltm, big[:, :, off:off + 8990 - off], scores, 6)
    check(ltm, big.transpose(0, 1), scores.t().contiguous(), 4)


def test_same_results_again_and_captured(ltm):
    import torch
    g = torch.Generator().manual_seed(4)
    logits = torch.randn((3, 4, 30011), generator=g).cuda()
    scores = -torch.rand((3, 4), generator=g).cuda()
    a = ltm.beam_select(logits, scores, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = ltm.beam_select(logits, scores, 8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = ltm.beam_select(logits, scores, 8, stream=s)
    s.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for x, y, z in zip(a, b, c):
        assert torch.equal(x, y) and torch.equal(x, z)
