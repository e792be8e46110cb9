"""Channels that the argument blocks' 32-bit fields cannot hold are refused before anything is copied or launched."""
import pytest
import torch

from serving_testlib import DEV

pytestmark = pytest.mark.gpu


def test_more_channels_than_32_bits_hold():
    import kda_b200
    for channels in ((1 << 32) + 64, (1 << 30) + 8):
        x = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device=DEV).expand(1, 1, channels)
        pool = torch.zeros(1, 1, device=DEV).expand(1, channels)
        for call in (lambda: kda_b200.gated_scan(x, x), lambda: kda_b200.gated_scan_step(x, x, None, None, None, None, pool), lambda: kda_b200.group_norm(x, 1 << 22)):
            with pytest.raises(ValueError, match="channels"):
                call()
    x = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device=DEV).expand(1, 1, (1 << 32) + 64)
    with pytest.raises(ValueError, match="channels"):
        kda_b200.short_conv(x, x[0, 0, :, None].expand(-1, 4))
    with pytest.raises(ValueError, match="channels"):
        kda_b200.selective_scan(x, x, torch.zeros(1, 1, device=DEV).expand(x.shape[2], 1), x[..., None, :1], x[..., None, :1])
