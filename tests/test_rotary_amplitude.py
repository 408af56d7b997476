"""The rotation's amplitude is an fp32 number: others are refused by name, before any launch (no GPU needed)."""

import pytest
import torch

from late_interaction_kernels.encoder import rotary


@pytest.mark.parametrize("amplitude", [1e39, -1e39, 3.5e38, float("inf"), -float("inf"), float("nan")])
def test_amplitudes_past_fp32_are_refused(amplitude):
    q, f = torch.zeros(1, 2, 1, 8), torch.ones(4, dtype=torch.float64)
    with pytest.raises(ValueError, match="amplitude"):
        rotary(q, frequencies=f, amplitude=amplitude)


@pytest.mark.parametrize("amplitude", [3.4028234e38, -3.4028234e38, 1e-60, 0, 2])
def test_others_go_on(amplitude):
    with pytest.raises(RuntimeError, match="GPU"):
        rotary(torch.zeros(1, 2, 1, 8), frequencies=torch.ones(4, dtype=torch.float64), amplitude=amplitude)


@pytest.mark.gpu
def test_the_largest_amplitude():
    q = torch.full((1, 2, 1, 8), 0.5, device="cuda")
    y = rotary(q, frequencies=torch.zeros(4, dtype=torch.float64, device="cuda"), amplitude=torch.finfo(torch.float32).max)
    assert torch.equal(y, torch.full_like(q, torch.finfo(torch.float32).max / 2))
