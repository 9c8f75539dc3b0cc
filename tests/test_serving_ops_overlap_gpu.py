"""Tree attention's output in the query's memory: as the query itself, or refused (more
than 512 sequences are several launches, and a later one would read what an earlier one
wrote)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [3, 600])
def test_output_in_the_querys_memory(ltm, B):
    import torch
    T, h, d, P = 2, 2, 64, 8
    buf = torch.randn((B + 1, T, h, d), device="cuda").half()
    k, v = (torch.randn((B, h, P, d), device="cuda").half() for _ in range(2))
    n = torch.full((B,), 3, dtype=torch.int32, device="cuda")
    want = ltm.tree_attention(buf[:-1], k, v, n)
    before = buf.clone()
    for q, out in ((buf[:-1], buf[1:]), (buf[1:], buf[:-1]),
                   (buf[:-1], buf[:-1].transpose(1, 2))):
        with pytest.raises(ltm.LtmError) as e:
            ltm.tree_attention(q, k, v, n, out=out)
        assert e.value.status == 1 and "overlap" in str(e.value)
    assert torch.equal(buf, before)
    ltm.tree_attention(buf[:-1], k, v, n, out=buf[:-1])
    assert torch.equal(buf[:-1], want)
    one = buf[:1, :1].clone()  # dimensions of one entry: any stride is the same
    same = torch.as_strided(one, one.shape, (7, 5, d, 1))
    want = ltm.tree_attention(one, k[:1], v[:1], n[:1])
    assert torch.equal(ltm.tree_attention(one, k[:1], v[:1], n[:1], out=same), want)
