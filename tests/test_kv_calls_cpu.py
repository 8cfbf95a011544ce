"""What the calls of the 4-bit KV cache refuse before any device work, and what their workspace is planned for: without a GPU."""
import pytest
import torch

from moelab_b200 import _lib, ops


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


def test_no_kernel_for_few_rows_where_no_row_fits_it():
    """More than 16 query heads per KV head: a call whose row tiles fill the GPU needs no workspace, with cu or without."""
    size = _lib.load().moeb_kv_attention_workspace_bytes  # T, B, P, page_size, H, kv_heads, head_dim, max_q, window, sinks, with_cu
    for cu in (0, 1):
        assert size(64, 64, 512, 64, 8 * 20, 8, 128, 1, 0, 0, cu) == 0
    assert size(128, 64, 512, 64, 8 * 16, 8, 128, 2, 0, 0, 0) == 0
    assert size(128, 64, 512, 64, 8 * 16, 8, 128, 2, 0, 0, 1) > 0  # some sequences may have one row: they fit
