"""Calls of the embedding, label and gradient operators at the edges of what their documentation allows."""
import pytest
import torch

from test_gpu_labels import _case

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------- label gradient
@pytest.mark.parametrize("rows,K", [(1, 9), (30, 9), (7, 300), (5, 5000)])
def test_label_gradients_that_come_lazily_negated(gpu_device, rows, K):
    """autograd hands on gradients that hold the other sign in memory, contiguous or not."""
    from gsplat.losses import label_log_probs

    dev = gpu_device
    x, y, g = _case(rows, K, torch.float32, rows + K)
    ups = [torch.randn(rows, generator=g).to(dev), torch.randn(rows, generator=g).to(dev), torch.randn(rows, 3, generator=g).to(dev)]

    def grad(up):
        leaf = x.to(dev).requires_grad_(True)
        got = label_log_probs(leaf, y.to(dev), top_k=3)
        return torch.autograd.grad([got.log_prob, got.entropy, got.top_log_probs], leaf, up)[0]

    want = grad([-u for u in ups])
    lazy = [torch._neg_view(u) for u in ups]
    assert all(u.is_neg() and u.is_contiguous() for u in lazy)
    assert torch.equal(grad(lazy), want)
    strided = [torch.complex(torch.zeros_like(u), u).conj().imag for u in ups]
    assert all(u.is_neg() for u in strided)
    assert torch.equal(grad(strided), want)
    # and as autograd makes them by itself
    leaf, plain = (x.to(dev).requires_grad_(True) for _ in range(2))
    lp = label_log_probs(leaf, y.to(dev)).log_prob
    torch.complex(torch.zeros_like(lp), lp).conj().imag.sum().backward()
    (-label_log_probs(plain, y.to(dev)).log_prob).sum().backward()
    assert torch.equal(leaf.grad, plain.grad)


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


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan"), -2.0])
@pytest.mark.parametrize("n,V,D", [(100, 50, 8), (256, 600, 3), (5000, 40, 16), (300_000, 64, 16), (5000, 90, 16), (300_000, 90, 16)])
def test_rows_that_no_id_selects_are_zeros_whatever_the_scale(gpu_device, n, V, D, scale):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    g = torch.Generator().manual_seed(n + V)
    ids = torch.randint(0, V, (n,), generator=g)
    ids[(ids % 3) == 1] = -1  # a third of the rows is selected by nothing
    up = torch.randn(n, D, generator=g)
    up[ids == 0] = 0.0  # a selected row whose sum is zero
    table = torch.zeros(V, D, device=dev, requires_grad=True)
    (v,) = torch.autograd.grad(embedding_lookup(table, ids.to(dev), scale), table, up.to(dev))
    v = v.cpu()
    none = torch.bincount(ids[ids >= 0], minlength=V) == 0
    assert bool(none.any()) and not bool(none.all())
    assert bool((v[none] == 0).all()) and not bool(torch.signbit(v[none]).any())
    if scale == -2.0:
        assert bool((v[0] == 0).all()) and bool((v[~none][1:] != 0).any())
    else:
        assert bool(torch.isnan(v[0]).all()) if not bool(none[0]) else True
        assert not bool(torch.isfinite(v[~none]).any())


# ------------------------------------------------------------------------------------------------- timing
def test_every_entry_point_is_timed(gpu_device):
    from gsplat import _backend as B
    from gsplat.gradients import clip_gradients, grad_norm
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(50, 12, device=dev, requires_grad=True)
    ids = torch.arange(5000, device=dev) % 50

    def step():
        out = embedding_lookup(table, ids)
        (v,) = torch.autograd.grad(label_log_probs(out, ids % 12, 2).log_prob.sum(), table)
        clip_gradients([v], 1.0)
        return grad_norm([v])

    want = step()
    names = {"gs_embedding_fwd", "gs_embedding_bwd", "gs_label_log_probs_fwd", "gs_label_log_probs_bwd", "gs_grad_clip", "gs_grad_norm"}
    B.profiling_start()
    try:
        step()
        assert torch.equal(step(), want)
    finally:
        seen = B.profiling_stop()
    assert set(seen) == names
    assert all(calls == 2 and 0.0 <= ms < 1e3 for calls, ms in seen.values()), seen
    B.profiling_start(only=["gs_label_log_probs_bwd"])
    step()
    assert set(B.profiling_stop()) == {"gs_label_log_probs_bwd"}
    step()
    assert B.profiling_stop() == {}
