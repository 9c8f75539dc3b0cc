"""The KV-cache and beam operators at the edges of what their callers may pass:
overlapping memory, dimensions of one entry, calls at once, captured calls."""
import pytest

pytestmark = pytest.mark.gpu


def refused(ltm, f):
    with pytest.raises(ltm.LtmError) as e:
        f()
    assert e.value.status == 1 and any(w in str(e.value) for w in ("overlap", "share"))


def test_overlapping_memory_is_refused(ltm):
    import torch
    B, h, P, d, T = 2, 2, 16, 64, 3
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    both = torch.zeros((2 * B * h * P * d + 8 * d,), device="cuda").half()
    one = both[:B * h * P * d].view(B, h, P, d)
    two = both[B * h * P * d:2 * B * h * P * d].view(B, h, P, d)
    late = both[8 * d:8 * d + B * h * P * d].view(B, h, P, d)
    k = torch.randn((B, T, h, d), device="cuda").half()
    before = both.clone()
    ltm.kv_cache_append(k[:, :0], k[:, :0], one, two, n)
    for kc, vc in ((one, one), (one, late), (late, two)):
        refused(ltm, lambda: ltm.kv_cache_append(k, k, kc, vc, n))
        refused(ltm, lambda: ltm.kv_cache_reorder([kc, vc], torch.zeros((1, B), dtype=torch.int32,
                                                                         device="cuda")))
    inside = one[:, :, 4:4 + T].transpose(1, 2)  # rows of the cache itself
    refused(ltm, lambda: ltm.kv_cache_append(inside, k, one, two, n))
    refused(ltm, lambda: ltm.kv_cache_append(k, inside, one, two, n))
    q8 = torch.zeros((B, h, P, d), dtype=torch.int8, device="cuda")
    s = torch.zeros((B, h, P), device="cuda")
    refused(ltm, lambda: ltm.kv_cache_append(k, k, q8, q8.clone(), n, s, s))
    refused(ltm, lambda: ltm.kv_cache_read(one, None, P, out=one))
    refused(ltm, lambda: ltm.tree_attention(k, one, two, n, out=one[:, :, :T].transpose(1, 2)))
    refused(ltm, lambda: ltm.tree_attention(k, one, two, n, out=k[:, :, :1].expand(k.shape)))
    torch.cuda.synchronize()
    assert torch.equal(both, before)
    # the output may be the query's own memory
    want = ltm.tree_attention(k, one, two, n)
    assert ltm.tree_attention(k, one, two, n, out=k).data_ptr() == k.data_ptr()
    assert torch.equal(k, want)


def test_dimensions_of_one_entry_have_no_stride(ltm):
    """PyTorch leaves the stride of a dimension of one entry open."""
    import torch
    h, P, d, V = 3, 40, 64, 50
    q = torch.randn((1, 1, h, d), device="cuda").half()
    kc, vc = (torch.randn((1, h, P, d), device="cuda").half() for _ in range(2))
    n = torch.full((1,), 20, dtype=torch.int32, device="cuda")
    odd = torch.as_strided(q, q.shape, (3, 1, d, 1))
    want_k, want_v = kc.clone(), vc.clone()
    ltm.kv_cache_append(q, q, want_k, want_v, n)
    ltm.kv_cache_append(odd, odd, kc, vc, n)
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    out = torch.as_strided(torch.empty_like(q), q.shape, (7, 5, d, 1))
    assert torch.equal(ltm.tree_attention(odd, kc, vc, n, out=out), ltm.tree_attention(q, kc, vc, n))
    x = torch.randn((1, 2, V, 4), device="cuda")[..., :1].squeeze(-1)[:, :, :1]  # V of one
    s = torch.tensor([[-1.0, -2.0]], device="cuda")
    got = ltm.beam_select(x, s)
    assert got[0].tolist() == [[-1.0, -2.0]] and got[1].tolist() == [[0, 1]]


@pytest.mark.parametrize("cache,T,G", [("same", 1, 1), ("int8", 1, 4), ("same", 20, 2),
                                       ("int8", 20, 2)])
def test_two_streams_at_once(ltm, cache, T, G):
    """Calls that run at the same time have their own workspaces."""
    import torch
    B, kvh, P, d = 2, 4, 3000, 64
    sets = []
    for i in range(2):
        g = torch.Generator().manual_seed(i)
        q = torch.randn((B, T, kvh * G, d), generator=g).half().cuda()
        k, v = (torch.randn((B, kvh, P, d), generator=g).half().cuda() for _ in range(2))
        ks = vs = None
        if cache == "int8":
            k, v = ((x * 40).clamp(-127, 127).to(torch.int8) for x in (k, v))
            ks, vs = (torch.rand((B, kvh, P), generator=g).cuda() * 0.02 for _ in range(2))
        n = torch.tensor([P - T - i, 100 + i], dtype=torch.int32, device="cuda")
        sets.append((q, k, v, n, None, ks, vs))
    want = [ltm.tree_attention(*a) for a in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            got[i].append(ltm.tree_attention(*sets[i], stream=st))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_two_captured_steps(ltm):
    """Two captured append + attend steps over one cache, replayed in turn while the
    lengths move on, against eager steps."""
    import torch
    B, T, kvh, G, P, d = 2, 10, 2, 3, 200, 128
    g = torch.Generator().manual_seed(9)

    def state():
        z = lambda *s, **kw: torch.zeros(s, device="cuda", **kw)
        return dict(k=z(B, kvh, P, d, dtype=torch.int8), v=z(B, kvh, P, d, dtype=torch.int8),
                    ks=z(B, kvh, P), vs=z(B, kvh, P), n=z(B, dtype=torch.int32))

    new = [torch.randn((B, T, kvh, d), generator=g).bfloat16().cuda() for _ in range(2)]
    q = [torch.randn((B, T, kvh * G, d), generator=g).bfloat16().cuda() for _ in range(2)]
    counts = torch.tensor([T, 4], dtype=torch.int32, device="cuda")

    def step(s, i):
        ltm.kv_cache_append(new[i], new[1 - i], s["k"], s["v"], s["n"], s["ks"], s["vs"], counts)
        o = ltm.tree_attention(q[i], s["k"], s["v"], s["n"], None, s["ks"], s["vs"], counts)
        s["n"].add_(counts)
        return o

    eager, other = state(), state()
    step(other, 0)
    graphs, outs = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, capture_error_mode="relaxed"):
            outs.append(step(other, i))
        graphs.append(gr)
    for x in other.values():
        x.zero_()
    for r in range(12):
        want = step(eager, r % 2)
        graphs[r % 2].replay()
        assert torch.equal(outs[r % 2], want), r
    for x in eager:
        assert torch.equal(eager[x], other[x]), x
    assert ltm.device_error() == 0
