"""weight_grad takes fp16 gradients with blocks of fp16 rows only: the values of bf16 and fp32 blocks may not fit fp16."""
import pytest
import torch

import self_forcing_amd as sfa

l8 = sfa.linear8


@pytest.mark.parametrize("dy", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [torch.bfloat16, torch.float16, torch.float32])
def test_mixed_types_are_refused(monkeypatch, dy, rows):
    def reached(*args):
        raise InterruptedError
    monkeypatch.setattr(l8, "_rows", reached)
    x8 = l8.Rows8(torch.zeros((4, 128), dtype=torch.uint8), torch.zeros(128, dtype=torch.uint8), (1, 4, 128), rows)
    fits = dy == torch.bfloat16 or rows == torch.float16
    with pytest.raises(InterruptedError if fits else ValueError, match=None if fits else "whose range"):
        l8.weight_grad(torch.zeros((1, 4, 8), dtype=dy), x8)
