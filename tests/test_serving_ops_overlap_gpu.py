"""Tree attention's output in the query's memory, as the query itself and shifted (more than
512 sequences are several launches, and a later one must not read what an earlier one
wrote)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [3, 600])
@pytest.mark.parametrize("other_stream", [False, True])
def test_output_in_the_querys_memory(ltm, B, other_stream):
    import torch
    T, h, d, P = 2, 2, 64, 8
    first = torch.randn((B + 1, T, h, d), device="cuda").half()
    k, v = (torch.randn((B, h, P, d), device="cuda").half() for _ in range(2))
    n = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream() if other_stream else torch.cuda.current_stream()
    for src, dst in ((slice(0, -1), slice(1, None)), (slice(1, None), slice(0, -1)),
                     (slice(0, -1), slice(0, -1))):
        want = ltm.tree_attention(first[src], k, v, n)
        buf = first.clone()
        torch.cuda.synchronize()
        out = buf[dst]
        assert ltm.tree_attention(buf[src], k, v, n, out=out, stream=stream) is out
        stream.synchronize()
        assert torch.equal(out, want)
    buf = first.clone()
    out = buf[:-1].transpose(1, 2)
    want = ltm.tree_attention(first[:-1], k, v, n)
    ltm.tree_attention(buf[:-1], k, v, n, out=out)
    assert torch.equal(out, want)
    one = first[:1, :1].clone()  # dimensions of one entry: any stride is the same
    same = torch.as_strided(one, one.shape, (7, 5, d, 1))
    want = ltm.tree_attention(one, k[:1], v[:1], n[:1])
    assert torch.equal(ltm.tree_attention(one, k[:1], v[:1], n[:1], out=same), want)


def test_columns_of_one_buffer(ltm):
    """Query and output as columns of the same rows: their spans meet, their elements do not."""
    import torch
    B, T, h, d, P = 520, 2, 2, 64, 8
    rows = torch.randn((B, T, 2, h, d), device="cuda").half()
    k, v = (torch.randn((B, h, P, d), device="cuda").half() for _ in range(2))
    n = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    q = rows[:, :, 0].clone()
    want = ltm.tree_attention(q, k, v, n)
    for b in (B, 4):
        ltm.tree_attention(rows[:b, :, 0], k[:b], v[:b], n[:b], out=rows[:b, :, 1])
        assert torch.equal(rows[:b, :, 1], want[:b]) and torch.equal(rows[:b, :, 0], q[:b])
