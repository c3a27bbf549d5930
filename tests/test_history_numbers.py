"""Numbers that do not fit the C structures' 32 bits are refused, not cut off."""
import numpy as np
import pytest


@pytest.mark.parametrize("kw", [dict(rotated=(1 << 32) + 32), dict(span=(1 << 32) + 64), dict(head_dim=(1 << 32) + 64), dict(rotated=32.0),
                                dict(original_length=(1 << 32) + 4096, scaling="yarn", factor=4.0), dict(rotated=-(1 << 32))])
def test_rotary(kw):
    from hydra_amd import history as hi
    with pytest.raises(ValueError):
        hi.Rotary(**{"head_dim": 64, "device": "cpu", **kw})
    assert hi.Rotary(np.int64(64), rotated=np.int32(32), span=64, device="cpu").turns.numel() == 16


@pytest.mark.parametrize("pinned", [(1 << 32) + 3, -(1 << 32), 2.0])
def test_histories(pinned):
    import torch
    from hydra_amd import history as hi
    k, n = torch.zeros((2, 3, 10, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        hi.History(k, k.clone(), n, ring=True, pinned=pinned)
    with pytest.raises(ValueError):
        hi.History.empty(2, 3, 10, 64, ring=True, pinned=pinned, device="cpu")
    assert hi.History(k, k.clone(), n, ring=True, pinned=np.int64(3)).c.pinned == 3


@pytest.mark.parametrize("tokens", [(1 << 32) + 1, 1.0, None])
def test_advances(tokens, monkeypatch):
    """Before anything of a device is asked for."""
    import torch
    from hydra_amd import history as hi
    monkeypatch.setattr(hi, "_cuda", lambda ctx, device: None)
    monkeypatch.setattr(hi, "lib", lambda: pytest.fail("reached the library"))
    h = hi.History.empty(2, 3, 10, 64, device="cpu")
    with pytest.raises(ValueError):
        hi.history_advance(None, h, torch.zeros(2, dtype=torch.int32), tokens)
