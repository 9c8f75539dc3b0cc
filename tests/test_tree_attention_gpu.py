"""Tree attention over a KV cache (ltm_tree_attention) on the GPU against a plain
evaluation in 64 bits.

Tolerance of an output element: the probabilities are rounded to 16 bits before
the value product (half a step u_p relative each: 2^-8 for bf16 products, 2^-11 for
f16, which int8 caches use too), so |error| <= u_p * A with A = sum_j p_j |v_j|;
the fp32 scores (|sum| of q k / sqrt(D) below 64 here, D products) and the
exponentials add less than 2^-12 * A; the output's own rounding adds u_o * |o|."""
import math

import numpy as np
import pytest

from _util import torch_dtype

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def quantised(x):
    """fp32 [..., d] -> (int8 codes, fp32 scales) in plain torch."""
    import torch
    s = x.abs().amax(-1)
    s = s / torch.full_like(s, 127.0)
    q = torch.round(x / torch.where(s == 0, torch.ones_like(s), s)[..., None]).clamp(-127, 127)
    return q.to(torch.int8), s


def reference(q, k, v, lens, num, parents):
    """64-bit outputs and A = sum p |v|; k, v: [B, kvh, P, d] values (double)."""
    import torch
    B, T, heads, d = q.shape
    G = heads // k.shape[1]
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    a = torch.zeros_like(o)
    for b in range(B):
        n = lens[b]
        for t in range(num[b]):
            at, x = [], t
            while x >= 0:
                at.append(n + x)
                x = x - 1 if parents is None else int(parents[b][x])
            idx = torch.tensor(list(range(n)) + at, device=q.device)
            kk, vv = k[b][:, idx].double(), v[b][:, idx].double()
            qq = q[b, t].double().reshape(-1, G, d)
            p = torch.softmax(qq @ kk.transpose(1, 2) / math.sqrt(d), -1)
            o[b, t] = (p @ vv).reshape(heads, d)
            a[b, t] = (p @ vv.abs()).reshape(heads, d)
    return o, a


def make(B, T, heads, kvh, d, P, dt, cache, lens, seed, scale=1.0):
    """q, caches (garbage behind every sequence's last token), and their values."""
    import torch
    g = torch.Generator().manual_seed(seed)
    td = torch_dtype(dt)
    q = torch.randn((B, T, heads, d), generator=g).to(td).cuda()
    k = (torch.randn((B, kvh, P, d), generator=g) * scale).to(td).cuda()
    v = torch.randn((B, kvh, P, d), generator=g).to(td).cuda()
    ks = vs = None
    if cache == "int8":
        k, ks = quantised(k.float())
        v, vs = quantised(v.float())
        vk, vv = k.double() * ks.double()[..., None], v.double() * vs.double()[..., None]
    else:
        vk, vv = k.double(), v.double()
    for b in range(B):  # never to be read into a result
        end = lens[b] + T
        if cache == "int8":
            ks[b, :, end:] = float("nan")
            vs[b, :, end:] = float("inf")
        else:
            k[b, :, end:] = float("nan")
            v[b, :, end:] = float("inf")
    return q, k, v, ks, vs, vk, vv


def tree(B, T, seed):
    rng = np.random.default_rng(seed)
    return [[max(-1, t - int(rng.integers(1, 5))) for t in range(T)] for _ in range(B)]


def check(got, o, a, dt, cache, what=""):
    import torch
    u_p = U["f16"] if cache == "int8" else U[dt]
    bound = a * (u_p + 2.0 ** -12) + U[dt] * o.abs() + 1e-30
    err = (got.double() - o).abs()
    assert torch.isfinite(got).all(), what
    bad = err > bound
    assert not bad.any(), (what, int(bad.sum()), float((err / bound).max()))


SHAPES = [  # B, T, heads, kvh, d, lens (None: spread up to this)
    (1, 1, 1, 1, 64, [0]), (1, 1, 1, 1, 128, [1]), (2, 1, 4, 4, 64, [127, 128]),
    (3, 1, 8, 2, 128, [129, 0, 300]), (2, 5, 12, 12, 64, [301, 17]), (1, 64, 1, 1, 128, [200]),
    (2, 64, 4, 2, 64, [0, 513]), (2, 13, 8, 1, 128, [1000, 64]), (1, 3, 64, 1, 64, [257]),
    (1, 17, 2, 2, 128, [255]), (4, 2, 2, 2, 64, [5, 383, 384, 385]), (1, 33, 3, 3, 64, [2000]),
]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("cache", ["same", "int8"])
@pytest.mark.parametrize("B,T,heads,kvh,d,lens", SHAPES)
def test_tree_matches_reference(ltm, dt, cache, B, T, heads, kvh, d, lens):
    import torch
    P = max(lens) + T + 3
    q, k, v, ks, vs, vk, vv = make(B, T, heads, kvh, d, P, dt, cache, lens, 7 * T + heads)
    par = tree(B, T, T)
    num = [T - (b % 2) for b in range(B)]
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ltm.tree_attention(q, k, v, torch.tensor(lens, **i32), torch.tensor(par, **i32), ks, vs,
                             num_tokens=torch.tensor(num, **i32))
    o, a = reference(q, vk, vv, lens, num, par)
    check(got, o, a, dt, cache)
    for b in range(B):
        assert not got[b, num[b]:].any(), "tokens a sequence does not have get zeros"
    got = ltm.tree_attention(q, k, v, torch.tensor(lens, **i32), k_scale=ks, v_scale=vs)  # a chain
    o, a = reference(q, vk, vv, lens, [T] * B, None)
    check(got, o, a, dt, cache, "chain")
    assert ltm.device_error() == 0


@pytest.mark.parametrize("dt,cache,T,G,d", [("bf16", "int8", 9, 2, 128), ("f16", "int8", 16, 4, 64),
                                           ("bf16", "int8", 64, 1, 64), ("f16", "int8", 11, 6, 128),
                                           ("f16", "same", 8, 4, 128), ("bf16", "same", 40, 3, 64),
                                           ("f16", "same", 22, 4, 64), ("f16", "same", 25, 4, 128),
                                           ("bf16", "same", 64, 4, 128), ("f16", "int8", 64, 2, 128)])
def test_many_rows_over_a_long_context(ltm, dt, cache, T, G, d):
    """18 to 256 rows per cached head with contexts cut over many CTAs: keys that grow
    towards the end (the references rise), V scales that span 2^6, query heads of very
    different sizes.  Scores have a deviation of at most 1, so that of a row's p * scale
    only those below 2^-14 of the largest (f16: 2^-25 off, not a relative 2^-11) make up
    less than that share of the sum: check's bound holds as it is."""
    import torch
    B, kvh = 3, 4
    lens = [12345, 0, 777]
    P = max(lens) + T + 5
    q, k, v, ks, vs, vk, vv = make(B, T, kvh * G, kvh, d, P, dt, cache, lens, 31 * T + G)
    mag = 2.0 ** (6 * torch.arange(kvh * G, device="cuda") / (kvh * G) - 7)
    q = (q.float() * mag[None, None, :, None]).to(q.dtype)
    rise = torch.linspace(0.25, 2.0, P, device="cuda")[None, None, :]
    size = 2.0 ** (6 * torch.rand((B, kvh, P), generator=torch.Generator().manual_seed(3)).cuda()
                   - 3).round()
    for b in range(B):
        e = lens[b] + T
        if cache == "int8":
            ks[b, :, :e] = (ks[b] * rise[0])[:, :e]
            vs[b, :, :e] = (vs[b] * size[b])[:, :e]
            vk[b, :, :e] = (k[b].double() * ks[b].double()[..., None])[:, :e]
            vv[b, :, :e] = (v[b].double() * vs[b].double()[..., None])[:, :e]
        else:
            k[b, :, :e] = (vk[b].float() * rise[0][..., None]).to(k.dtype)[:, :e]
            vk[b, :, :e] = k[b, :, :e].double()
    par = tree(B, T, 2)
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ltm.tree_attention(q, k, v, torch.tensor(lens, **i32), torch.tensor(par, **i32), ks, vs)
    o, a = reference(q, vk, vv, lens, [T] * B, par)
    check(got, o, a, dt, cache)


@pytest.mark.parametrize("cache", ["same", "int8"])
def test_long_context_over_many_ctas(ltm, cache):
    """Contexts long enough that several CTAs share a head, next to empty and
    short sequences; scores that grow along the context (the reference maximum is
    raised again and again) and that fall."""
    import torch
    B, T, h, d, dt = 5, 3, 2, 128, "bf16"
    lens = [20000, 0, 9999, 128, 31]
    P = max(lens) + T
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, P, dt, cache, lens, 5)
    ramp = torch.linspace(0, 6, P, device="cuda")
    for b, sign in ((0, 1.0), (2, -1.0)):
        # keys drift along the first token's query: scores from 0 to 6 |q|^2 / sqrt(d)
        add = sign * ramp[None, :, None] * q[b, 0, :, None, :].float() / math.sqrt(d) * 4
        end = lens[b] + T
        val = (vk[b].float() + add).to(torch_dtype(dt))
        if cache == "int8":
            kq, sq = quantised(val.float())
            k[b, :, :end], ks[b, :, :end] = kq[:, :end], sq[:, :end]
            vk[b] = kq.double() * sq.double()[..., None]
        else:
            k[b, :, :end] = val[:, :end]
            vk[b] = val.double()
    par = tree(B, T, 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ltm.tree_attention(q, k, v, torch.tensor(lens, **i32), torch.tensor(par, **i32), ks, vs)
    o, a = reference(q, vk, vv, lens, [T] * B, par)
    check(got, o, a, dt, cache)


def test_value_scales_of_any_ratio(ltm):
    """int8 value rows whose scales span 40 powers of two, the largest where the
    probability is smallest, and an all-zero row: the small ones still count."""
    import torch
    B, T, h, d, dt, n = 1, 2, 2, 64, "bf16", 400
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, n + T, dt, "int8", [n], 11)
    e = torch.arange(n + T, device="cuda") % 41 - 20
    # scores fall by 1 (a factor of e) per power of two that the scale rises
    kv = q[0, 0].float()[:, None] * (-e.float()[None, :, None]) * math.sqrt(d) \
        / (q[0, 0].float() ** 2).sum(-1)[:, None, None]
    kq, sq = quantised(kv)
    k[0], ks[0] = kq, sq
    vs[0] = vs[0] * torch.exp2(e.float())
    vs[0, :, 7] = 0
    v[0, :, 7] = 0
    vk = k.double() * ks.double()[..., None]
    vv = v.double() * vs.double()[..., None]
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ltm.tree_attention(q, k, v, torch.tensor([n], **i32), None, ks, vs)
    o, a = reference(q, vk, vv, [n], [T], None)
    check(got, o, a, dt, "int8")


def test_query_magnitudes_with_int8_keys(ltm):
    """bf16 queries far outside f16's range against int8 keys of the inverse scale."""
    import torch
    B, T, h, d, n = 1, 3, 2, 128, 150
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, n + T, "bf16", "int8", [n], 12)
    f = torch.tensor([2.0 ** 60, 2.0 ** -60, 1.0], device="cuda")
    q = (q.float() * f[None, :, None, None]).bfloat16()
    q[0, 2] = 0
    for t in range(2):
        s = ks / f[t]
        got = ltm.tree_attention(q, k, v, torch.tensor([n], dtype=torch.int32, device="cuda"),
                                 None, s, vs)
        o, a = reference(q, k.double() * s.double()[..., None], vv, [n], [T], None)
        check(got[:, t:t + 1], o[:, t:t + 1], a[:, t:t + 1], "bf16", "int8")
        check(got[:, 2:], o[:, 2:], a[:, 2:], "bf16", "int8")


def test_non_finite_values_stay_where_they_are_seen(ltm):
    """A NaN / infinite value or key of one draft branch reaches the tokens below
    it and no other; a NaN in the context reaches every token of its sequence."""
    import torch
    B, T, h, d, dt = 2, 6, 2, 64, "f16"
    lens = [140, 9]
    par = [[-1, 0, 0, 1, 2, -1], [-1, 0, 1, 2, 3, 4]]
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, 160, dt, "same", lens, 3)
    i32 = dict(dtype=torch.int32, device="cuda")
    args = (torch.tensor(lens, **i32), torch.tensor(par, **i32))
    clean = ltm.tree_attention(q, k, v, *args)
    v[0, :, lens[0] + 1] = float("inf")
    k[0, :, lens[0] + 5] = float("nan")
    v[1, :, 4] = float("nan")
    got = ltm.tree_attention(q, k, v, *args)
    for t in (0, 2, 4):
        assert torch.equal(got[0, t], clean[0, t])
    for t in (1, 3):
        assert not torch.isfinite(got[0, t]).any()
    assert torch.isnan(got[0, 5]).all()
    assert torch.isnan(got[1]).all()


@pytest.mark.parametrize("dt,cache,G,d", [("f16", "same", 4, 64), ("bf16", "same", 12, 128),
                                         ("bf16", "same", 21, 64), ("bf16", "int8", 2, 128),
                                         ("f16", "int8", 4, 64)])
def test_non_finite_drafts_with_more_rows(ltm, dt, cache, G, d):
    """The same with 12 to 126 rows per cached head, and with int8 rows whose scale is NaN
    (what the append makes of a non-finite row)."""
    import torch
    B, T, kvh = 2, 6, 2
    lens = [126, 300]  # the first draft crosses a tile
    par = [[-1, 0, 0, 1, 2, -1]] * 2
    q, k, v, ks, vs, vk, vv = make(B, T, kvh * G, kvh, d, 310, dt, cache, lens, 13)
    i32 = dict(dtype=torch.int32, device="cuda")
    args = (torch.tensor(lens, **i32), torch.tensor(par, **i32), ks, vs)
    clean = ltm.tree_attention(q, k, v, *args)
    for b in range(B):
        if cache == "int8":
            vs[b, :, lens[b] + 1] = float("nan")
            ks[b, :, lens[b] + 5] = float("nan")
        else:
            v[b, :, lens[b] + 1, ::3] = float("-inf")
            v[b, :, lens[b] + 1, 1::3] = float("nan")
            v[b, :, lens[b] + 1, 2::3] = float("inf")
            k[b, :, lens[b] + 5] = float("inf")
            k[b, :, lens[b] + 5, 0] = float("nan")
    got = ltm.tree_attention(q, k, v, *args)
    for t in (0, 2, 4):
        assert torch.equal(got[:, t], clean[:, t])
    for t in (1, 3):
        assert not torch.isfinite(got[:, t]).any()
    assert torch.isnan(got[:, 5]).all()


def test_bad_lengths_and_parents(ltm):
    import torch
    B, T, h, d, dt = 4, 3, 2, 64, "bf16"
    lens = [10, 10, 10, 10]
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, 20, dt, "same", lens, 4)
    i32 = dict(dtype=torch.int32, device="cuda")
    got = ltm.tree_attention(q, k, v, torch.tensor([10, 18, -1, 10], **i32),
                             num_tokens=torch.tensor([3, 3, 3, 4], **i32))
    torch.cuda.synchronize()
    assert ltm.device_error() == 5
    assert not got[1:].any()
    o, a = reference(q, vk, vv, lens, [T, 0, 0, 0], None)
    check(got[:1], o[:1], a[:1], dt, "same")
    # a parent that is the token itself, a later one, or below -1: counts as a root
    bad = [[0, 0, 1], [-1, 2, 0], [-5, 0, 0], [-1, 0, 1]]
    fixed = [[-1, 0, 1], [-1, -1, 0], [-1, 0, 0], [-1, 0, 1]]
    got = ltm.tree_attention(q, k, v, torch.tensor(lens, **i32), torch.tensor(bad, **i32))
    torch.cuda.synchronize()
    assert ltm.device_error() == 7
    o, a = reference(q, vk, vv, lens, [T] * B, fixed)
    check(got, o, a, dt, "same")


def test_strided_operands_streams_and_out(ltm):
    """q as columns of fused rows, an output with strides of its own, another stream."""
    import torch
    B, T, h, d, dt = 2, 4, 3, 64, "f16"
    lens = [33, 150]
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, 160, dt, "same", lens, 6)
    fused = torch.zeros((B, T, 3, h, d), dtype=q.dtype, device="cuda")
    fused[:, :, 0] = q
    out = torch.full((B, h, T, d), 3.0, dtype=q.dtype, device="cuda").transpose(1, 2)
    lt = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = ltm.tree_attention(fused[:, :, 0], k, v, lt, out=out, stream=s)
    s.synchronize()
    assert got is out
    o, a = reference(q, vk, vv, lens, [T] * B, None)
    check(out, o, a, dt, "same")


def test_captured_and_replayed(ltm):
    """One graph, replayed while the lengths and the cache move on the device."""
    import torch
    B, T, h, d, dt = 2, 2, 4, 128, "bf16"
    P = 600
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, P, dt, "int8", [P - T] * B, 9)
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    ltm.tree_attention(q, k, v, lens, k_scale=ks, v_scale=vs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ltm.tree_attention(q, k, v, lens, k_scale=ks, v_scale=vs)
    for n in ([0, 5], [128, 127], [598, 300], [1, 0]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        graph.replay()
        o, a = reference(q, vk, vv, n, [T] * B, None)
        check(got, o, a, dt, "int8")
        assert torch.equal(got, ltm.tree_attention(q, k, v, lens, k_scale=ks, v_scale=vs))


def test_many_sequences(ltm):
    """More sequences than one launch takes."""
    import torch
    B, T, h, d, dt = 1030, 1, 1, 64, "f16"
    lens = [(b * 7) % 40 for b in range(B)]
    q, k, v, ks, vs, vk, vv = make(B, T, h, h, d, 41, dt, "same", lens, 2)
    got = ltm.tree_attention(q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    o, a = reference(q, vk, vv, lens, [T] * B, None)
    check(got, o, a, dt, "same")


@pytest.mark.parametrize("cache", ["same", "int8"])
def test_offsets_beyond_32_bits(ltm, cache):
    """A cache of more than 2^31 elements; only its last sequence is looked at."""
    import torch
    B, T, h, d, dt, P = 8, 1, 32, 128, "f16", 70000
    td = torch.int8 if cache == "int8" else torch_dtype(dt)
    k = torch.zeros((B, h, P, d), dtype=td, device="cuda")
    v = torch.zeros_like(k)
    ks = vs = None
    n = 1000
    q, k1, v1, ks1, vs1, vk, vv = make(1, T, h, h, d, n + T, dt, cache, [n], 8)
    k[-1, :, :n + T], v[-1, :, :n + T] = k1[0], v1[0]
    if cache == "int8":
        ks, vs = torch.zeros((B, h, P), device="cuda"), torch.zeros((B, h, P), device="cuda")
        ks[-1, :, :n + T], vs[-1, :, :n + T] = ks1[0], vs1[0]
    qq = torch.zeros((B, T, h, d), dtype=q.dtype, device="cuda")
    qq[-1] = q[0]
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens[-1] = n
    got = ltm.tree_attention(qq, k, v, lens, k_scale=ks, v_scale=vs)
    o, a = reference(q, vk, vv, [n], [T], None)
    check(got[-1:], o, a, dt, cache)


@pytest.mark.parametrize("dt,cache", [("bf16", "int8"), ("f16", "same")])
def test_draft_verify_append_run(ltm, dt, cache):
    """The operators as a server uses them: prompts appended, then rounds of
    appending a draft tree, attending it, and re-appending the accepted branch's
    rows in order; every round equals the 64-bit reference on the values that the
    cache reads back."""
    import torch
    B, T, h, kvh, d, P = 2, 7, 4, 2, 64, 96
    td = torch_dtype(dt)
    g = torch.Generator().manual_seed(5)
    i32 = dict(dtype=torch.int32, device="cuda")
    ct = torch.int8 if cache == "int8" else td
    kc = torch.zeros((B, kvh, P, d), dtype=ct, device="cuda")
    vc = torch.zeros_like(kc)
    ks = torch.zeros((B, kvh, P), device="cuda") if cache == "int8" else None
    vs = torch.zeros((B, kvh, P), device="cuda") if cache == "int8" else None
    rand = lambda *s: torch.randn(s, generator=g).to(td).cuda()  # noqa: E731
    prompt = [40, 23]
    ltm.kv_cache_append(rand(B, 40, kvh, d), rand(B, 40, kvh, d), kc, vc, torch.zeros(B, **i32), ks,
                        vs, torch.tensor(prompt, **i32))
    lens = list(prompt)
    for rnd in range(3):
        par = tree(B, T, rnd)
        k, v, q = rand(B, T, kvh, d), rand(B, T, kvh, d), rand(B, T, h, d)
        lt = torch.tensor(lens, **i32)
        ltm.kv_cache_append(k, v, kc, vc, lt, ks, vs)
        got = ltm.tree_attention(q, kc, vc, lt, torch.tensor(par, **i32), ks, vs)
        vk = ltm.kv_cache_read(kc, ks, P).double()
        vv = ltm.kv_cache_read(vc, vs, P).double()
        o, a = reference(q, vk, vv, lens, [T] * B, par)
        check(got, o, a, dt, cache, f"round {rnd}")
        path = []  # the accepted branch: the last token's ancestors, in order
        for b in range(B):
            x, p = T - 1, []
            while x >= 0:
                p.append(x)
                x = par[b][x]
            path.append(p[::-1])
        n = [len(p) for p in path]
        pad = torch.tensor([p + [0] * (T - len(p)) for p in path], device="cuda")
        rows = torch.arange(B, device="cuda")[:, None]
        ltm.kv_cache_append(k[rows, pad], v[rows, pad], kc, vc, lt, ks, vs, torch.tensor(n, **i32))
        lens = [a_ + b_ for a_, b_ in zip(lens, n)]
    assert ltm.device_error() == 0
