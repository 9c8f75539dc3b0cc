"""A call on a stream other than the current one: its outputs must not lie in memory that
work still queued on the current stream uses."""
import pytest

pytestmark = pytest.mark.gpu


def _calls(ltm):
    """name -> (call on a stream, bytes of the output that is looked at)."""
    import torch
    B, h, P, d = 4, 8, 1024, 128
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((B, h, P, d), generator=g).half().cuda() for _ in range(2))
    q = torch.randn((B, 40, 4 * h, d), generator=g).half().cuda()
    n = torch.full((B,), P - 64, dtype=torch.int32, device="cuda")
    logits = torch.randn((64, 4, 1000), generator=g).cuda()
    scores = torch.zeros((64, 4), device="cuda")
    return {"read": (lambda s: ltm.kv_cache_read(k, None, 900, stream=s), B * h * 900 * d * 2),
            "tree": (lambda s: ltm.tree_attention(q, k, v, n, stream=s), q.numel() * 2),
            "beam": (lambda s: ltm.beam_select(logits, scores, 60, stream=s)[0], 64 * 60 * 4)}


@pytest.mark.parametrize("what", ["read", "tree", "beam"])
def test_memory_freed_with_work_pending(ltm, what):
    import torch
    call, size = _calls(ltm)[what]
    other = torch.cuda.Stream()
    want = call(None).clone()
    call(other)  # the other stream's pool has its blocks
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    for _ in range(3):
        x = torch.full((size,), 7, dtype=torch.uint8, device="cuda")
        y = torch.zeros_like(x)
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)  # about 50 ms
        y.copy_(x)
        del x
        got = call(other)
        other.synchronize()
        torch.cuda.synchronize()
        assert (y == 7).all(), "the call wrote into memory that the current stream still reads"
        assert torch.equal(got, want)
        del got, y


@pytest.mark.parametrize("what", ["read", "tree", "beam"])
def test_output_dropped_while_the_current_stream_reads_it(ltm, what):
    """The output of a call on another stream, read on the current one (which waits for
    it) and dropped before that read has run: the next call must not get its memory."""
    import torch
    call, _ = _calls(ltm)[what]
    other = torch.cuda.Stream()
    want = call(None).clone()
    copy = torch.empty_like(want)
    for _ in range(3):
        torch.cuda.synchronize()
        out = call(other)
        torch.cuda.current_stream().wait_stream(other)
        torch.cuda._sleep(100_000_000)
        copy.copy_(out)
        del out
        with torch.cuda.stream(other):
            junk = [torch.full_like(want, 3) for _ in range(2)]
        other.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(copy, want)
        del junk


@pytest.mark.parametrize("what", ["read", "tree", "beam"])
def test_captured_on_a_branch(ltm, what):
    """A call on a stream that joined a capture, replayed while the inputs stay; outputs of
    two calls do not share memory."""
    import torch
    call, _ = _calls(ltm)[what]
    want = call(None).clone()
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        here = torch.cuda.current_stream()
        other.wait_stream(here)
        a = call(other)
        b = call(None)
        here.wait_stream(other)
        c = a.clone()
        d = call(None)
    for _ in range(3):
        for x in (a, b, c, d):
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in (a, b, c, d))
