"""Histories that `History.empty` makes: their zeros are filled on torch's stream, which a context's does not wait for."""
import pytest


def test_on_the_host():
    import torch
    from hydra_amd import history as hi
    for fmt, width in (("f16", 64), ("bf16", 64), ("mxfp8", 64), ("mxfp4", 32)):
        h = hi.History.empty(2, 3, 5, 64, format=fmt, device="cpu")
        assert h.k.shape == h.v.shape == (2, 3, 5, width) and h.lengths.tolist() == [0, 0]
        assert all(t is None or not t.any() for t in (h.k, h.v, h.k_scales, h.v_scales))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["mxfp8", "bf16"])
@pytest.mark.parametrize("own_stream", [False, True])
def test_complete_when_returned(fmt, own_stream):
    """Behind much work on torch's stream, and written at once."""
    import torch
    from hydra_amd import history as hi
    from hydra_amd.layer import Context
    ctx = Context(0)
    k, v = (torch.randn((2, 3, 2, 64), device="cuda:0").bfloat16() for _ in range(2))
    counts = torch.full((2,), 3, dtype=torch.int32, device="cuda:0")
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    x = torch.ones((8192, 8192), dtype=torch.bfloat16, device="cuda:0")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream() if own_stream else torch.cuda.current_stream()
    with torch.cuda.stream(stream):
        for _ in range(20):
            torch.mm(x, x, out=y)
        h = hi.History.empty(2, 2, 100000, 64, format=fmt)
        assert stream.query()
        hi.history_write(ctx, h, k, v, counts)
        hi.history_read_into(ctx, h, h.lengths, counts, ko, vo)
    ctx.synchronize()
    torch.cuda.synchronize()
    assert h.lengths.tolist() == [0, 0] and not h.k[:, :, 3:].any() and not h.v[:, :, 3:].any()
    if fmt == "bf16":
        assert torch.equal(ko, k) and torch.equal(vo, v)
    else:   # within half a step of the 32 columns' scale: at most 2^-4 of a group's largest
        for a, b in ((ko, k), (vo, v)):
            top = b.float().view(2, 3, 2, 2, 32).abs().amax(-1, keepdim=True).expand(2, 3, 2, 2, 32).reshape(b.shape)
            assert ((a.float() - b.float()).abs() <= top / 16).all()
