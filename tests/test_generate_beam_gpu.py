"""TitanModel.generate_beam (decode step, beam_select and kv_cache_reorder in a
captured step) against a plain beam search that uses the model's own decode step,
64-bit log-softmax and copied caches."""
import pytest

from test_generate_gpu import _model

pytestmark = pytest.mark.gpu


def plain_beam(ltm, model, prompt, n, W, end):
    import torch
    B, S = prompt.shape
    V = model.vocab
    seqs, out_scores = [], []
    for b in range(B):
        cache = model.make_cache(W, S + n)
        _, lg = model.prefill(prompt[b:b + 1].expand(W, S).contiguous(), cache)
        lp = torch.log_softmax(lg[:1].double(), -1)
        best, x = torch.sort(lp[0], descending=True, stable=True)
        scores, toks = best[:W].clone(), [[int(t)] for t in x[:W]]
        done = [t[0] == end for t in toks]
        for i in range(1, n):
            tok = torch.tensor([t[-1] for t in toks], dtype=torch.int32, device="cuda")
            lens = torch.full((W,), S + i - 1, dtype=torch.int32, device="cuda")
            lg = model.decode_step(tok, lens, cache)
            # the scores that the step continues from are stored as fp32
            tot = scores.float().double()[:, None] + torch.log_softmax(lg.double(), -1)
            for w in range(W):
                if done[w]:
                    tot[w] = -float("inf")
                    tot[w, end] = float(scores[w])
            best, flat = torch.sort(tot.flatten(), descending=True, stable=True)
            rows = [int(f) // V for f in flat[:W]]
            new = [int(f) % V for f in flat[:W]]
            scores = best[:W].clone()
            toks = [toks[r] + [t] for r, t in zip(rows, new)]
            done = [done[r] or t == end for r, t in zip(rows, new)]
            for c in cache._k + cache._v:
                c.copy_(c[rows])
        seqs.append(toks)
        out_scores.append(scores)
    return torch.tensor(seqs, dtype=torch.int32), torch.stack(out_scores)


@pytest.mark.parametrize("scheme,dt", [("w8a8", "bf16"), ("w4a16", "bf16"), ("w8a8", "f16")])
@pytest.mark.parametrize("W,end", [(4, None), (3, 17), (1, None)])
def test_beam_search_matches_plain(ltm, orc, scheme, dt, W, end):
    import torch
    from ltm_b200 import synthetic
    V, B, S, N = 1000, 2, 21, 7
    model, *_ = _model(ltm, scheme, dt, V=V, seed=3)
    prompt = torch.from_numpy(synthetic.tokens(B, S, V, 5)).cuda()
    if end is not None:  # an end token that the search does meet
        end = int(model.generate_beam(prompt, 3, W, use_graph=False)[0][0, 0, 1])
    toks, scores = model.generate_beam(prompt, N, W, end_token=end)
    again, scores2 = model.generate_beam(prompt, N, W, end_token=end, use_graph=False)
    assert torch.equal(toks, again) and torch.equal(scores, scores2)
    want, ws = plain_beam(ltm, model, prompt, N, W, -1 if end is None else end)
    # a step adds at most 5e-6 (the fp32 sum of exponentials) and the rounding of the stored
    # score (2^-24 of it): N steps
    assert (scores.cpu().double() - ws.cpu()).abs().max() <= N * (5e-6 + 2.0 ** -24 * ws.abs().max())
    assert torch.equal(toks.cpu(), want)
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    if W == 1:
        greedy, _ = model.generate_greedy(prompt, N)
        assert torch.equal(toks[:, 0], greedy)
    if end is not None:
        hit = (toks == end).int().cummax(-1).values.bool()
        assert bool(hit.any()) and bool((toks[hit] == end).all())
    assert ltm.device_error() == 0
    model.close()


def test_beam_search_refuses_bad_sizes(ltm):
    import torch
    model, *_ = _model(ltm, "w8a8", "bf16", V=100)
    prompt = torch.zeros((1, 8), dtype=torch.int32, device="cuda")
    for args in ((0, 2), (4, 0)):
        with pytest.raises(ltm.LtmError):
            model.generate_beam(prompt, *args)
    with pytest.raises(ltm.LtmError):
        model.generate_beam(prompt, 8, 2, max_positions=10)
    toks, scores = model.generate_beam(prompt, 1, 5)
    assert toks.shape == (1, 5, 1) and len(set(toks.flatten().tolist())) == 5
    model.close()
