"""Calls of the embedding, label and gradient operators at the edges of what their documentation allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------- embedding gradient
@pytest.mark.parametrize("D", [0, 1, 16, 128, 129])
@pytest.mark.parametrize("n", [0, 1, 256, 257, 5000, 20_000])
def test_a_table_without_rows(gpu_device, n, D):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.zeros(0, D, device=dev, requires_grad=True)
    out = embedding_lookup(table, torch.arange(n, device=dev) - 3, 2.0)
    assert out.shape == (n, D) and bool((out == 0).all())
    out.sum().backward()
    assert table.grad.shape == (0, D)
