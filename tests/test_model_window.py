"""A window of the model's attention has at least one position, with either attention; first tokens that stay visible are not a negative number of them."""
import pytest

from tirocinio_triennale_b200.models import GPT2, GPT2Config


@pytest.mark.parametrize("fused,attention", [(False, "torch"), (True, "torch"), (True, "own")])
@pytest.mark.parametrize("bad", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(sinks=-1)])
def test_refused(bad, fused, attention):
    cfg = GPT2Config.tiny()
    cfg.fused, cfg.attention = fused, attention
    for name, value in bad.items():
        setattr(cfg, name, value)
    with pytest.raises(ValueError, match="window|sinks"):
        GPT2(cfg)


def test_smallest_window():
    import torch

    cfg = GPT2Config.tiny()
    cfg.window = 1
    idx = torch.randint(0, 257, (2, 32), generator=torch.Generator().manual_seed(0))
    assert GPT2(cfg)(idx, idx).isfinite()
