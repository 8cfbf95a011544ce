"""What the calls of the 4-bit KV cache refuse before any device work, and what their workspace is planned for: without a GPU."""
import pytest
import torch

from moelab_b200 import ops


class Fake:
    device, index, kv_heads, head_dim = torch.device("cuda", 0), 0, 2, 64


def test_tensors_that_need_gradients_are_refused():
    plain = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    grad = plain.clone().requires_grad_()
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    calls = [lambda t: ops.kv_write(Fake, t, plain, table, lens), lambda t: ops.kv_attention(t, Fake, table, lens)]
    for call in calls:
        with pytest.raises(ValueError, match="backward"):
            call(grad)
        with pytest.raises(ValueError, match="CUDA"):  # as far as any CPU tensor comes
            call(grad.detach())
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call(grad)
