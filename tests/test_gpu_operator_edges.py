"""Calls of the embedding, label and gradient operators at the edges of what their documentation allows, and sums whose
every partial sum is exact, so that a row left out anywhere shows."""
import pytest
import torch

from operator_bounds import assert_within, rounding
from test_gpu_labels import _case, _check, _reference

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


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


def _exact_sums(ids, values, V):
    """Sums of integer rows in 64 bits, over the ids in [0, V): differences of the running sums of the sorted rows."""
    keep = (ids >= 0) & (ids < V)
    s, order = ids[keep].sort()
    run = torch.nn.functional.pad(values[keep][order].double().t().contiguous().cumsum(1), (1, 0))
    cut = torch.searchsorted(s, torch.arange(V + 1, device=ids.device))
    return (run[:, cut[1:]] - run[:, cut[:-1]]).t()


def _whole_rows(n, D, dtype, dev):
    """Values of -2 to 2: with a power of two as the scale every sum of up to 2^22 of them is exact in fp32, in any order."""
    assert n <= 1 << 22
    up = torch.randint(-2, 3, (n, D), generator=torch.Generator(device=dev).manual_seed(n), device=dev).to(dtype)
    up[:, 0] = 1.0  # a count: no two rows can stand in for each other
    return up


def _check_exact(name, ids, V, up):
    from gsplat.prepass import embedding_lookup

    table = torch.zeros(V, up.shape[1], device=up.device, dtype=up.dtype, requires_grad=True)
    (v,) = torch.autograd.grad(embedding_lookup(table, ids, 0.5), table, up)
    want = (_exact_sums(ids, up, V) * 0.5).float().to(up.dtype)
    assert torch.equal(v, want), f"{name}: {int((v != want).sum())} of {v.numel()} differ"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,D", [(257, 64, 1), (5000, 1, 128), (300_000, 64, 16), (300_000, 3, 5), (1_000_000, 8, 100),
                                   (16_384, 70, 20), (16_385, 70, 20), (40_000, 5000, 24), (70_001, 300, 33), (300_000, 65, 16),
                                   (131_072, 70_000, 8), (100_003, 1000, 704), (20_000, 7, 300), (5000, 1, 256), (66_000, 1 << 20, 2),
                                   (1_000_000, 200_000, 16), (1_000_001, 65, 7)])
@pytest.mark.parametrize("kind", ["uniform", "grouped", "few", "one", "outside"])
def test_no_row_is_left_out_of_a_sum(gpu_device, n, V, D, dtype, kind):
    g = torch.Generator().manual_seed(n + V)
    if kind == "one":
        ids = torch.full((n,), V - 1, dtype=torch.int64)
    elif kind == "few":
        ids = torch.randint(0, 3, (n,), generator=g) * (V // 3)
    else:
        ids = torch.randint(0, V, (n,), generator=g)
    if kind == "grouped":
        ids = ids.sort().values
    elif kind == "outside":
        ids[torch.rand(n, generator=g) < 0.5] = -1
    _check_exact(f"{dtype} {n}x{V}x{D} {kind}", ids.to(gpu_device), V, _whole_rows(n, D, dtype, gpu_device))


@pytest.mark.parametrize("n,V,D", [(4000, 100, 16), (40_000, 100, 16), (140_000, 70, 3), (140_000, 300, 64), (20_000, 500, 260),
                                   (60_000, 90, 1200), (1_200_000, 100, 16)])
def test_no_row_is_left_out_of_a_long_run(gpu_device, n, V, D):
    """Runs that start and end anywhere in what one workgroup has, up to all ids but a few."""
    dev = gpu_device
    g, up = torch.Generator(device=dev).manual_seed(n + D), _whole_rows(n, D, torch.float32, dev)
    for lead in (0, 1, 15, 64, 257, 1024, 4097):
        for length in (16, 17, 63, 64, 65, 256, 257, 511, 1024, 1500, 4096, 8191, n // 2, n - 3000, n - lead - 1, n - lead):
            if length < 1 or lead + length > n:
                continue
            ids = torch.full((n,), V - 1, device=dev)
            ids[:lead] = torch.arange(lead, device=dev) % (V // 3)
            ids[lead:lead + length] = V // 2
            rest = n - lead - length
            ids[lead + length:] = V // 2 + 1 + torch.arange(rest, device=dev) % (V - V // 2 - 1)
            ids = ids[torch.randperm(n, generator=g, device=dev)]
            _check_exact(f"run of {length} behind {lead} of {n}x{V}x{D}", ids, V, up)


def test_values_behind_32_bits(gpu_device):
    """The gradient of a table of more than 2^31 elements: every row that was selected, and nothing else."""
    from gsplat.prepass import embedding_lookup

    dev, V, D = gpu_device, 1_100_000, 2048
    table = torch.zeros(V, D, device=dev, dtype=torch.bfloat16, requires_grad=True)
    rows = torch.tensor([V - 1, 0, V - 2], device=dev)
    out = embedding_lookup(table, rows.repeat(200))
    (v,) = torch.autograd.grad(out, table, torch.ones_like(out))
    assert bool((v[rows] == 200).all())
    assert sorted((v != 0).any(1).nonzero()[:, 0].tolist()) == sorted(rows.tolist())


# ------------------------------------------------------------------------------------------------- alternatives
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [66, 100, 129, 160, 200, 255, 299, 511])
@pytest.mark.parametrize("top", [9, 17, 21, 32, 33, 64])
def test_many_alternatives_of_middling_rows(gpu_device, K, top, dtype):
    """More of them than lanes that hold values, in rows of ordinary values."""
    x, y, _ = _case(37, K, dtype, K + top)
    _check(f"{dtype} 37x{K} top {top}", gpu_device, x, y, top=top)


@pytest.mark.parametrize("rows,K,dtype,top", [(2_000_003, 19, torch.float32, 3), (2_000_003, 63, torch.bfloat16, 2),
                                              (40_001, 1001, torch.float32, 5), (80_000, 1999, torch.bfloat16, 33),
                                              (300, 120_001, torch.float32, 64), (2000, 40_001, torch.float16, 8)])
def test_large_gradients_with_alternatives(gpu_device, rows, K, dtype, top):
    """Gradients that are stored past the caches, with the alternatives' terms stored behind them."""
    from gsplat.losses import label_log_probs

    dev = gpu_device
    g = torch.Generator(device=dev).manual_seed(rows)
    x = (torch.randn(rows, K, device=dev, generator=g) * 3).to(dtype).requires_grad_(True)
    y = torch.randint(-1, K, (rows,), device=dev, generator=g)
    ups = [torch.randn(rows, device=dev, generator=g), torch.randn(rows, device=dev, generator=g), torch.randn(rows, top, device=dev, generator=g)]
    got = label_log_probs(x, y, top)
    (v,) = torch.autograd.grad([got.log_prob, got.entropy, got.top_log_probs], x, ups)
    some = torch.cat([torch.arange(4), torch.randint(0, rows, (8,)), torch.arange(rows - 4, rows)]).to(dev)
    ref = _reference(x.detach()[some], y[some], top, *(u[some] for u in ups))
    assert torch.equal(got.top_labels[some].cpu(), ref["top_labels"])
    assert_within(f"{rows}x{K} {dtype} v", v[some], ref["v"][0], ref["v"][1] + rounding(dtype, ref["v"][0]))


def test_saved_tensors_that_travel_and_graphs_that_stay(gpu_device):
    """What the backward needs may be kept elsewhere meanwhile; a graph can be walked twice; no graph is made where none is."""
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(700, 40, device=dev, requires_grad=True)
    ids = torch.randint(-1, 700, (9000,), device=dev)
    render = torch.randn(9000, 60, device=dev, requires_grad=True)

    def step():
        got = label_log_probs(embedding_lookup(table, ids) + render[:, 7:47], ids % 40, 4)
        return got.log_prob.sum() + got.entropy.sum() + got.top_log_probs.sum(), got

    def sliced():
        got = label_log_probs(render[:, 3:43], ids % 40, 4)
        return got.log_prob.sum() + got.top_log_probs.sum(), got

    for make, leaves in ((step, [table, render]), (sliced, [render])):
        loss, got = make()
        want = torch.autograd.grad(loss, leaves, retain_graph=True)
        again = torch.autograd.grad(loss, leaves)
        assert all(torch.equal(a, b) for a, b in zip(want, again))
        with torch.autograd.graph.save_on_cpu():
            loss, _ = make()
        assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(loss, leaves)))
        with torch.inference_mode():
            _, plain = make()
        assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(got, plain))


def test_long_sort_and_alternatives_in_a_graph(gpu_device):
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev, n, V, D = gpu_device, 40_000, 3000, 130
    table = torch.randn(V, D, device=dev, requires_grad=True)
    ids, up = torch.randint(0, V, (n,), device=dev), torch.randn(n, 40, device=dev)

    def step():
        got = label_log_probs(embedding_lookup(table, ids, 0.5), ids % D, 40)
        return [got.log_prob, got.top_labels, torch.autograd.grad([got.log_prob, got.top_log_probs], table, [up[:, 0], up])[0]]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        with torch.no_grad():
            table.normal_(), up.normal_(), ids.random_(-1, V + 1)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), k


# ------------------------------------------------------------------------------------------------- clipping
@pytest.mark.parametrize("inplace", [False, True])
def test_a_captured_clip_within_and_beyond_the_limit(gpu_device, inplace):
    from gsplat.gradients import clip_gradients

    dev = gpu_device
    raw = [torch.randn(n, device=dev).to(t) for n, t in ((50_001, torch.float32), (3, torch.bfloat16), (4099, torch.float16))]
    work = [t.clone() for t in raw]
    clip_gradients([t.clone() for t in raw], 1.0, inplace=inplace)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, norm = clip_gradients(work, 1.0, inplace=inplace)
    for k, scale in enumerate((1e-4, 1.0, 1e-3, 30.0, 1e-4)):
        for t, w in zip(raw, work):
            t.normal_().mul_(scale)
            w.copy_(t)
        want, n = clip_gradients(raw, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert (float(n) < 1.0) == (scale < 1e-2), (k, float(n))
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(captured, want)), k
        if scale < 1e-2:
            assert all(torch.equal(a, b) for a, b in zip(captured, raw)), k


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
