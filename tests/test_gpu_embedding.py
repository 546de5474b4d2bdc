"""gsplat.prepass.embedding_lookup (gs_embedding_fwd / _bwd) against its formula in 64 bits.

Bounds: the output is one fp32 product (U) and one rounding; a row of the gradient is an fp32 sum of c terms in some order
(c U sum|x|), one product and one rounding (operator_bounds.py)."""
import pytest
import torch

from operator_bounds import U, assert_within, rounding

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ids(kind, n, V, g):
    if kind == "one":  # all the same
        return torch.full((n,), V // 2, dtype=torch.int64)
    if kind == "few":
        return torch.randint(0, min(V, 3), (n,), generator=g)
    ids = torch.randint(0, V, (n,), generator=g)
    if kind == "grouped":
        ids = ids.sort().values
    if kind == "outside":  # a third selects nothing, on both sides and far away
        bad = torch.rand(n, generator=g) < 0.33
        ids[bad] = torch.tensor([-1, V, -(2 ** 31), 2 ** 31 - 1, V + 7])[torch.randint(0, 5, (int(bad.sum()),), generator=g)]
    return ids


def _reference(table, ids, scale, v_out):
    """(out, v_table, sum of |terms| per entry, count per row) in 64 bits."""
    V, D = table.shape
    ok = (ids >= 0) & (ids < V)
    out = torch.zeros(ids.shape[0], D, dtype=torch.float64)
    out[ok] = table.double()[ids[ok]] * scale
    v, a = torch.zeros(V, D, dtype=torch.float64), torch.zeros(V, D, dtype=torch.float64)
    v.index_add_(0, ids[ok], v_out.double()[ok])
    a.index_add_(0, ids[ok], v_out.double()[ok].abs())
    return out, v * scale, a * abs(scale), torch.bincount(ids[ok], minlength=V).double()


def _check(name, dev, table, ids, scale, v_out, **kw):
    from gsplat.prepass import embedding_lookup

    t = table.to(dev).requires_grad_(True)
    out = embedding_lookup(t, ids.to(dev), scale, **kw)
    (v,) = torch.autograd.grad(out, t, v_out.to(dev))
    assert out.dtype == table.dtype and v.dtype == table.dtype and v.shape == table.shape
    scale = float(torch.tensor(scale, dtype=torch.float32))
    r_out, r_v, r_abs, count = _reference(table, ids.long(), scale, v_out)
    assert_within(name + " out", out, r_out, r_out.abs() * U + rounding(table.dtype, r_out))
    assert_within(name + " v_table", v, r_v, (count[:, None] + 1) * U * r_abs + rounding(table.dtype, r_v))
    assert bool((v[(count == 0).to(dev)] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 600, 48), (5, 7, 3), (256, 31, 17), (257, 31, 17), (64, 5, 130), (65, 5, 513),
                                   (1000, 300, 1), (3000, 1000, 5), (4097, 129, 64), (9000, 64, 16), (20011, 5000, 12),
                                   (700, 3, 2050), (2049, 257, 1000)])
@pytest.mark.parametrize("kind", ["uniform", "grouped", "one", "few", "outside"])
def test_against_the_formula(gpu_device, dtype, n, V, D, kind):
    g = torch.Generator().manual_seed(n * 7 + V + D)
    table, v_out = torch.randn(V, D, generator=g).to(dtype), torch.randn(n, D, generator=g).to(dtype)
    _check(f"{dtype} {n}x{V}x{D} {kind}", gpu_device, table, _ids(kind, n, V, g), 1.7, v_out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,V,D", [(16384, 70, 20), (16385, 70, 20), (40_000, 5000, 24), (70_001, 300, 33), (300_000, 64, 16),
                                   (300_000, 65, 16), (300_000, 3, 5), (131_072, 70_000, 8), (100_003, 1000, 704), (20_000, 7, 300),
                                   (257, 64, 1), (5000, 1, 256), (66_000, 1 << 20, 2), (17_000, 300_000, 1)])
@pytest.mark.parametrize("kind", ["uniform", "grouped", "skewed", "one", "outside"])
def test_many_ids(gpu_device, dtype, n, V, D, kind):
    """Every sort, the form for few rows, and both lengths of a piece."""
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    g = torch.Generator().manual_seed(n + V + D)
    ids = torch.randint(0, V, (n,), generator=g)
    if kind == "grouped":
        ids = ids.sort().values
    elif kind == "skewed":
        ids = (torch.rand(n, generator=g) ** 8 * V).long().clamp_(max=V - 1)
    elif kind == "one":
        ids = torch.full_like(ids, V - 1)
    elif kind == "outside":
        ids = torch.where(torch.rand(n, generator=g) < 0.5, torch.randint(-3, V + 4, (n,), generator=g), -1)
    table = torch.randn(V, D, generator=g).to(dtype).to(dev).requires_grad_(True)
    up = torch.randn(n, D, generator=g).to(dtype)
    (v,) = torch.autograd.grad(embedding_lookup(table, ids.to(dev), 0.25), table, up.to(dev))
    row = torch.where((ids >= 0) & (ids < V), ids, torch.full_like(ids, V))
    ref, size = (torch.zeros(V + 1, D, dtype=torch.float64).index_add_(0, row, t)[:V] * 0.25 for t in (up.double(), up.double().abs()))
    count = torch.bincount(row, minlength=V + 1)[:V].double()
    assert_within(f"{dtype} {n}x{V}x{D} {kind}", v, ref, (count[:, None] + 1) * U * size + rounding(dtype, ref))
    assert bool((v[(count == 0).to(dev)] == 0).all())


@pytest.mark.parametrize("n", [0, 63, 64, 65, 128, 129, 255, 300, 4096, 4160])
def test_run_lengths_around_the_pieces(gpu_device, n):
    """Runs that end at, before and behind the pieces a long run is cut into, next to short ones."""
    g = torch.Generator().manual_seed(n)
    runs = [torch.full((m,), k) for k, m in enumerate((n, 1, 64, 65, 63, 2, 129, 0, n, 64))]
    ids = torch.cat(runs)[torch.randperm(sum(len(r) for r in runs), generator=g)]
    table, v_out = torch.randn(11, 33, generator=g), torch.randn(len(ids), 33, generator=g)
    _check(f"runs {n}", gpu_device, table, ids, 1.0, v_out)
    for short in (15, 16, 17, 31, 32, 33):  # and pieces of 16, in a table too large for the form for few rows
        runs = [torch.full((m,), 7 * k) for k, m in enumerate((n, 1, short, 1, short + 1, 15, 16, 17, short, 47, 48, 49, 2))]
        ids = torch.cat(runs)[torch.randperm(sum(len(r) for r in runs), generator=g)]
        table, v_out = torch.randn(97, 9, generator=g), torch.randn(len(ids), 9, generator=g)
        _check(f"runs {n} {short}", gpu_device, table, ids, 1.0, v_out)


def test_strides_shapes_types_and_alignment(gpu_device):
    from gsplat.prepass import embedding_lookup

    dev, g = gpu_device, torch.Generator().manual_seed(3)
    wide = torch.randn(50, 41, generator=g)
    for cols in (slice(0, 16), slice(1, 17), slice(3, 40), slice(0, 41, 2)):  # a slice of columns: a row stride of 41
        table = wide.to(dev)[:, cols].requires_grad_(True)
        ids = torch.randint(0, 50, (3, 4, 5), generator=g, dtype=torch.int32)
        out = embedding_lookup(table, ids.to(dev), -2.0)
        assert out.shape == (3, 4, 5, table.shape[1])
        assert torch.equal(out.cpu(), wide[:, cols][ids.long()] * -2.0)
        up = torch.randn(5, 4, 3, table.shape[1], generator=g).to(dev).permute(2, 1, 0, 3)  # not contiguous
        (v,) = torch.autograd.grad(out, table, up)
        ref = torch.zeros(50, table.shape[1], dtype=torch.float64).index_add_(
            0, ids.long().reshape(-1), up.double().cpu().reshape(60, -1)) * -2.0
        assert_within(f"strided {cols}", v, ref, 60 * U * 60 * ref.abs().max() + 1e-12)
    table = wide.to(dev).requires_grad_(True)
    ids = torch.randint(0, 50, (600, 2), generator=g).to(dev)
    out = embedding_lookup(table, ids[:, 1])  # every other id
    assert torch.equal(out.cpu(), wide[ids[:, 1].cpu()])
    out.sum().backward()  # a broadcast gradient
    assert torch.equal(table.grad.cpu(), torch.bincount(ids[:, 1].cpu(), minlength=50).float()[:, None].expand(50, 41))
    t3 = wide.to(dev)[:1].expand(9, 41)  # rows that share memory
    assert torch.equal(embedding_lookup(t3, ids[:, 0] % 9).cpu(), wide[:1].expand(600, 41))


def test_empty_sides(gpu_device):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    for V, D, n in ((4, 3, 0), (0, 3, 5), (4, 0, 5), (0, 0, 0)):
        t = torch.randn(V, D, device=dev, requires_grad=True)
        out = embedding_lookup(t, torch.zeros(n, dtype=torch.int64, device=dev))
        assert out.shape == (n, D) and bool((out == 0).all() if V == 0 else True)
        out.sum().backward()
        assert t.grad.shape == (V, D) and bool((t.grad == (n if V > 0 else 0) * (torch.arange(V, device=dev)[:, None] == 0)).all())


def test_special_values_stay_in_their_rows(gpu_device):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(300, 8, device=dev)
    table[5], table[6] = float("nan"), float("inf")
    t = table.clone().requires_grad_(True)
    ids = torch.arange(3000, device=dev) % 300
    out = embedding_lookup(t, ids, 3.0)
    assert torch.equal(torch.isnan(out).any(1), ids == 5) and torch.equal(torch.isinf(out).any(1), ids == 6)
    up = torch.ones(3000, 8, device=dev)
    up[307] = float("nan")
    up[ids == 9] = torch.finfo(torch.float32).max / 4
    (v,) = torch.autograd.grad(out, t, up)
    assert torch.equal(torch.isnan(v).any(1).nonzero()[:, 0].cpu(), torch.tensor([7]))
    assert bool(torch.isinf(v[9]).all()) and bool((v[0] == 30.0).all())


def test_same_bits_on_every_run_and_stream(gpu_device):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    g = torch.Generator(device=dev).manual_seed(1)
    table = torch.randn(1000, 24, device=dev, generator=g).requires_grad_(True)
    ids = (torch.rand(200_000, device=dev, generator=g) ** 6 * 1000).long()
    up = torch.randn(200_000, 24, device=dev, generator=g)
    first = torch.autograd.grad(embedding_lookup(table, ids), table, up)[0]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        second = torch.autograd.grad(embedding_lookup(table, ids), table, up)[0]
    torch.cuda.current_stream(dev).wait_stream(side)
    assert torch.equal(first, second)
    assert torch.equal(first, torch.autograd.grad(embedding_lookup(table, ids.int()), table, up)[0])


@pytest.mark.parametrize("n,V,D", [(7, 600, 48), (5000, 64, 16), (5000, 3000, 40)])
def test_captured_and_replayed(gpu_device, n, V, D):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(V, D, device=dev).requires_grad_(True)
    ids, up = torch.randint(0, V, (n,), device=dev), torch.randn(n, D, device=dev)

    def step():
        out = embedding_lookup(table, ids, 0.5)
        return out, torch.autograd.grad(out, table, up)[0]

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
        assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1]), k


def test_offsets_behind_32_bits(gpu_device):
    """A table and an output of more than 2^31 elements: the last rows are the right ones."""
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    V, D = 1_100_000, 2048
    table = torch.zeros(V, D, device=dev, dtype=torch.bfloat16)
    table[-2:] = torch.randn(2, D, device=dev).bfloat16()
    table.requires_grad_(True)
    ids = torch.tensor([V - 1, 0, V - 2] * 200, device=dev)
    out = embedding_lookup(table, ids)
    assert torch.equal(out[::3], table.detach()[-1:].expand(200, D)) and torch.equal(out[2::3], table.detach()[-2:-1].expand(200, D))
    up = torch.ones_like(out)
    (v,) = torch.autograd.grad(out, table, up)
    assert bool((v[-2:] == 200).all()) and bool((v[0] == 200).all())
    assert float(v.float().sum()) == 600.0 * D if False else int((v != 0).any(1).sum()) == 3
    del table, out, v, up
    small = torch.randn(3, D, device=dev, dtype=torch.float32).bfloat16().requires_grad_(True)
    n = 1_100_000
    ids = torch.arange(n, device=dev) % 3
    out = embedding_lookup(small, ids)
    assert torch.equal(out[-3:], small.detach()[ids[-3:]])
    up = torch.zeros(n, D, device=dev, dtype=torch.bfloat16)
    up[-1] = 1.5
    (v,) = torch.autograd.grad(out, small, up)
    assert bool((v[int(ids[-1])] == 1.5).all()) and int((v != 0).any(1).sum()) == 1


def test_refusals_on_the_device(gpu_device):
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    t, ids = torch.randn(4, 3, device=dev), torch.zeros(2, dtype=torch.int64, device=dev)
    with pytest.raises(IndexError):
        embedding_lookup(t, ids + 4, validate=True)
    with pytest.raises(IndexError):
        embedding_lookup(t, ids - 1, validate=True)
    embedding_lookup(t, ids + 3, validate=True)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding_lookup(t, ids.cpu())
    leaf = t.clone().requires_grad_(True)
    (v,) = torch.autograd.grad(embedding_lookup(leaf, ids).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        v.sum().backward()


@pytest.mark.parametrize("n", [100, 256])
def test_few_ids_of_one_row(gpu_device, n):
    g = torch.Generator().manual_seed(n)
    table, v_out = torch.randn(500, 24, generator=g), torch.randn(n, 24, generator=g)
    _check(f"one row {n}", gpu_device, table, torch.full((n,), 77), 1.0, v_out)


@pytest.mark.parametrize("n", [0, 1, 200])
def test_few_ids_on_a_large_table(gpu_device, n):
    from gsplat.prepass import embedding_lookup

    dev, V, D = gpu_device, 70_000, 1001
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(-1, V, (n,), generator=g)
    ids[n // 2 :] = V - 1
    up = torch.randn(n, D, generator=g)
    table = torch.zeros(V, D, device=dev, requires_grad=True)
    (v,) = torch.autograd.grad(embedding_lookup(table, ids.to(dev), 2.0), table, up.to(dev))
    rows, where = torch.unique(ids[ids >= 0], return_inverse=True)
    ref, size = (torch.zeros(len(rows), D, dtype=torch.float64).index_add_(0, where, t[ids >= 0]) * 2.0 for t in (up.double(), up.double().abs()))
    assert_within(f"large {n}", v[rows.to(dev)], ref, (n + 1) * U * size + rounding(torch.float32, ref))
    assert set((v != 0).any(1).nonzero()[:, 0].tolist()) == set(rows.tolist())


def test_two_threads_on_streams_of_their_own(gpu_device):
    import threading

    from gsplat.gradients import clip_gradients
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(4000, 40, device=dev)
    ids = [torch.randint(0, 4000, (30_000,), device=dev) for _ in range(2)]

    def step(k):
        t = table.clone().requires_grad_(True)
        got = label_log_probs(embedding_lookup(t, ids[k], 2.0), ids[k] % 40, top_k=3)
        (v,) = torch.autograd.grad(got.log_prob.sum(), t)
        clipped, norm = clip_gradients([v], 0.5)
        return [got.log_prob, got.top_labels, v, clipped[0], norm]

    want = [step(0), step(1)]
    torch.cuda.synchronize()
    seen = [[], []]

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream(dev)):
            for _ in range(10):
                seen[k].append(step(k))
            torch.cuda.current_stream(dev).synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(seen[k]) == 10
        assert all(torch.equal(a, b) for got in seen[k] for a, b in zip(got, want[k]))


def test_captured_backward_next_to_an_eager_graph_is_refused(gpu_device):
    """An eager graph of the same leaf, made on another stream and still alive, would pull that stream into the capture."""
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(20, 8, device=dev).requires_grad_(True)
    ids, labels = torch.arange(20, device=dev), torch.arange(20, device=dev) % 8
    for make in (lambda: embedding_lookup(table, ids).sum(), lambda: label_log_probs(table, labels).log_prob.sum()):
        make().backward()  # (warm)
        table.grad = None
        eager = make()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(graph):
                make().backward()
        eager.backward()
        assert bool(torch.isfinite(table.grad).all())
        table.grad = None
        del eager, graph


def test_captured_backward_behind_other_nodes_is_refused_too(gpu_device):
    """The leaf lies behind views and products here, or its gradient is asked for and not accumulated: an eager graph made
    on a stream of its own is in nobody's way then."""
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    table = torch.randn(2, 10, 8, device=dev).requires_grad_(True)
    ids, labels = torch.arange(20, device=dev), torch.arange(20, device=dev).view(2, 10) % 8
    for make in (lambda: embedding_lookup((table * 2.0).view(20, 8), ids).sum(), lambda: label_log_probs(table, labels).log_prob.sum()):
        make().backward()  # (warm)
        want, table.grad = table.grad, None
        eager = make()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(graph):
                make().backward()
        eager.backward()
        assert torch.equal(table.grad, want)
        table.grad = None
        eager = make()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph of the same leaf"):
            with torch.cuda.graph(graph):
                torch.autograd.grad(make(), table)
        del eager
        side = torch.cuda.Stream(dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            eager = make()
        torch.cuda.current_stream(dev).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(make(), table)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        del eager, graph, got


def test_negated_views(gpu_device):
    """Tensors that torch negates lazily hold the other sign in memory."""
    from gsplat.gradients import clip_gradients
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev = gpu_device
    x = torch.randn(30, 9, device=dev)
    neg = torch.complex(torch.zeros_like(x), x).conj().imag
    assert neg.is_neg() and torch.equal(neg, -x)
    plain = (-x).contiguous()
    ids, labels = torch.arange(20, device=dev) % 30, torch.arange(30, device=dev) % 9
    assert torch.equal(embedding_lookup(neg, ids), embedding_lookup(plain, ids))
    assert all(torch.equal(a, b) for a, b in zip(label_log_probs(neg, labels, 3), label_log_probs(plain, labels, 3)))
    (a,), norm_a = clip_gradients([neg], 0.5)
    (b,), norm_b = clip_gradients([plain], 0.5)
    assert torch.equal(a, b) and torch.equal(norm_a, norm_b)
    clip_gradients([neg], 0.5, inplace=True)
    assert torch.equal(neg, b)


@pytest.mark.parametrize("n,V,D", [(4000, 100, 16), (40_000, 100, 16), (140_000, 70, 3), (140_000, 300, 64), (20_000, 500, 260), (60_000, 90, 1200)])
def test_runs_as_long_as_several_workgroups(gpu_device, n, V, D):
    """Runs that start and end anywhere in what one workgroup has, from a few of its pieces to most of the ids: the sums of
    the gradient come from single pieces, whole workgroups and both."""
    from gsplat.prepass import embedding_lookup

    dev, g = gpu_device, torch.Generator().manual_seed(n + D)
    table, v_out = torch.zeros(V, D, device=dev).requires_grad_(True), torch.randn(n, D, generator=g)
    up, wide, size = v_out.to(dev), v_out.double(), v_out.double().abs()
    for lead in (0, 1, 15, 64, 257, 1024) if n * D < 10_000_000 else (0, 257):
        for length in (16, 63, 64, 65, 256, 257, 511, 1024, 1500, 4096, n - 3000, n - lead):
            if length < 1 or lead + length > n or (n * D > 10_000_000 and length < 256):
                continue
            ids = torch.full((n,), V - 1, dtype=torch.int64)
            ids[:lead] = torch.arange(lead) % (V // 3)
            ids[lead:lead + length] = V // 2
            rest = n - lead - length
            ids[lead + length:] = V // 2 + 1 + torch.arange(rest) % (V - V // 2 - 1)
            ids = ids[torch.randperm(n, generator=g)]
            (v,) = torch.autograd.grad(embedding_lookup(table, ids.to(dev)), table, up)
            want, terms = torch.zeros(V, D, dtype=torch.float64), torch.zeros(V, D, dtype=torch.float64)
            want.index_add_(0, ids, wide)
            terms.index_add_(0, ids, size)
            count = torch.bincount(ids, minlength=V)[:, None]
            assert_within(f"run of {length} behind {lead} of {n}x{V}x{D}", v, want, (count + 1) * U * terms + rounding(v.dtype, want))
