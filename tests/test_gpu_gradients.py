"""gsplat.gradients (gs_grad_norm / gs_grad_clip) against their formulas in 64 bits.

Bounds: the norm is a 64-bit sum and root, rounded once (U = 2^-24 of itself).  The factor has the norm, its sum with
1e-6, max_norm as fp32 and a division (4 U), the product one more, and the result one rounding."""
import pytest
import torch

from operator_bounds import U, assert_within, rounding

pytestmark = pytest.mark.gpu

MIX = [torch.float32, torch.bfloat16, torch.float16]


def _grads(sizes, dtypes, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=g) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def _norm(grads):
    return torch.stack([t.double().square().sum() for t in grads]).sum().sqrt()


def _check(name, dev, grads, max_norm, inplace):
    from gsplat.gradients import clip_gradients, grad_norm

    norm = _norm(grads)
    factor = min(1.0, max_norm / (float(norm) + 1e-6))
    mine = [t.to(dev) for t in grads]
    n0 = grad_norm(mine)
    got, n1 = clip_gradients(mine, max_norm, inplace=inplace)
    assert n0.shape == n1.shape == () and torch.equal(n0, n1)
    assert_within(name + " norm", n1, norm, norm * U * 1.001 + 1e-45)
    assert len(got) == len(grads)
    for i, (a, b, src) in enumerate(zip(got, grads, mine)):
        ref = b.double() * factor
        assert a.dtype == b.dtype and a.shape == b.shape and (a is src) == inplace
        assert_within(f"{name} [{i}]", a, ref, ref.abs() * 5 * U + rounding(b.dtype, ref))
        if not inplace:
            assert torch.equal(src.cpu(), b)
        if factor == 1.0 and float(norm) + 1e-6 < max_norm * (1 - 1e-6):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("max_norm", [0.0, 1e-3, 1.0, 1e9, float("inf")])
@pytest.mark.parametrize("sizes", [[1], [3], [8], [0, 5, 0], [7, 8, 9, 15, 16, 17], [1000, (33, 5), 1, (4, 4, 4)], [100_003, 31],
                                   [8192, 8193, 8191, 16384, 16385, 32769], list(range(1, 63)), [5] * 300, [2_000_003, 70_000, 9]])
def test_against_the_formula(gpu_device, sizes, max_norm, inplace):
    for dtypes in ([torch.float32], [torch.bfloat16], [torch.float16], MIX):
        _check(f"{len(sizes)} {dtypes[0]} {max_norm}", gpu_device, _grads(sizes, dtypes, len(sizes)), max_norm, inplace)


@pytest.mark.parametrize("tensors", [127, 128, 129, 256, 257, 700])
def test_more_tensors_than_a_launch_carries(gpu_device, tensors):
    _check(f"{tensors}", gpu_device, _grads([1 + i % 37 for i in range(tensors)], MIX, tensors), 0.5, True)
    _check(f"{tensors}", gpu_device, _grads([1 + i % 37 for i in range(tensors)], MIX, tensors), 0.5, False)


def test_alignment_strides_and_orders(gpu_device):
    from gsplat.gradients import clip_gradients

    dev = gpu_device
    for dtype in MIX:
        base = torch.randn(9, 5000, device=dev).to(dtype)
        flat = torch.randn(9 * 5001, device=dev).to(dtype)
        views = [flat[i * 5000 + i : (i + 1) * 5000 + i] for i in range(9)]  # starts at every alignment
        views += [base.t(), base[:, ::3][:4], torch.randn(3, 4, 5, 6, device=dev).to(dtype).permute(3, 1, 0, 2)]
        host = [v.cpu().clone() for v in views[:9]] + [v.cpu() for v in views[9:]]
        keep = base.clone()
        out, norm = clip_gradients(views, 1.0)
        ref_norm = _norm(host)
        assert_within("norm", norm, ref_norm, ref_norm * U * 1.001)
        for a, b in zip(out, host):
            ref = b.double() / (float(ref_norm) + 1e-6)
            assert_within("view", a, ref, ref.abs() * 5 * U + rounding(dtype, ref))
        assert torch.equal(base, keep)
        # in place through a view with gaps: what lies between is left as it was
        col = torch.randn(50, 7, device=dev).to(dtype)
        before = col.clone()
        clip_gradients([col[:, 2], col[:, 5]], 0.1, inplace=True)
        assert torch.equal(col[:, [0, 1, 3, 4, 6]], before[:, [0, 1, 3, 4, 6]])
        ref = before[:, [2, 5]].double() * (0.1 / (float(before[:, [2, 5]].double().norm()) + 1e-6))
        assert_within("columns", col[:, [2, 5]], ref.cpu(), ref.abs().cpu() * 5 * U + rounding(dtype, ref.cpu()))


def test_range_and_special_values(gpu_device):
    from gsplat.gradients import clip_gradients, grad_norm

    dev = gpu_device
    for v in (1e25, 1e-25, 3e38, 1e-38):  # squares far outside fp32
        g = torch.full((1000,), v, device=dev)
        want = float(g.double().norm())
        got = float(grad_norm([g]))
        assert (got == want if want == float("inf") else abs(got - want) <= want * U * 1.001) if want < 3.4e38 else got == float("inf")
    big = [torch.full((3,), 1e30, device=dev), torch.ones(5, device=dev, dtype=torch.bfloat16)]
    out, norm = clip_gradients(big, 1.0)
    assert abs(float(out[0].double().norm()) - 1.0) < 1e-6
    bad = [torch.tensor([1.0, float("nan")], device=dev), torch.ones(3, device=dev)]
    out, norm = clip_gradients(bad, 1.0)
    assert bool(torch.isnan(norm)) and all(bool(torch.isnan(t).all()) for t in out)
    inf = [torch.tensor([1.0, float("inf")], device=dev), torch.ones(3, device=dev)]
    out, norm = clip_gradients(inf, 1.0)
    assert float(norm) == float("inf") and out[1].tolist() == [0.0] * 3 and float(out[0][0]) == 0.0 and bool(torch.isnan(out[0][1]))
    keep = [t.clone() for t in inf]
    with pytest.raises(RuntimeError, match="not finite"):
        clip_gradients(inf, 1.0, inplace=True, error_if_nonfinite=True)
    assert all(torch.equal(a, b) for a, b in zip(inf, keep))
    zero = [torch.zeros(10, device=dev)]
    out, norm = clip_gradients(zero, 1.0, inplace=True, error_if_nonfinite=True)
    assert float(norm) == 0.0 and bool((out[0] == 0).all())


def test_parameters(gpu_device):
    from gsplat.gradients import clip_grad_norm

    dev = gpu_device
    p = [torch.nn.Parameter(torch.randn(n, 3, device=dev)) for n in (5, 100, 1)] + [torch.nn.Parameter(torch.randn(2, device=dev))]
    q = [torch.nn.Parameter(t.detach().clone()) for t in p]
    for a, b in zip(p[:3], q[:3]):
        a.grad = torch.randn_like(a)
        b.grad = a.grad.clone()
    ids = [id(t.grad) for t in p[:3]]
    n1 = clip_grad_norm((t for t in p + p[:1]), 0.7)  # a generator, one without a gradient, one named twice
    n2 = torch.nn.utils.clip_grad_norm_(q, 0.7)
    assert [id(t.grad) for t in p[:3]] == ids and p[3].grad is None
    assert abs(float(n1) - float(n2)) <= 1e-5 * float(n2)
    for a, b in zip(p[:3], q[:3]):
        assert torch.allclose(a.grad, b.grad, rtol=1e-5, atol=0)
    assert float(clip_grad_norm([p[3]], 1.0)) == 0.0
    assert float(clip_grad_norm(p[0], 1e9)) > 0


def test_same_bits_in_place_and_out_on_every_stream(gpu_device):
    from gsplat.gradients import clip_gradients

    dev = gpu_device
    grads = [t.to(dev) for t in _grads([1_000_003, 77, (300, 41)], MIX, 5)]
    a, na = clip_gradients(grads, 1.0)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        b, nb = clip_gradients(grads, 1.0)
    torch.cuda.current_stream(dev).wait_stream(side)
    version = grads[0]._version
    c, nc = clip_gradients(grads, 1.0, inplace=True)
    assert grads[0]._version > version
    assert torch.equal(na, nb) and torch.equal(na, nc)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


@pytest.mark.parametrize("inplace", [False, True])
def test_captured_and_replayed(gpu_device, inplace):
    from gsplat.gradients import clip_gradients

    dev = gpu_device
    raw = [torch.randn(n, device=dev).to(t) for n, t in ((50_001, torch.float32), (3, torch.bfloat16), (4099, torch.float16))]
    work = [t.clone() for t in raw]
    clip_gradients([t.clone() for t in raw], 1.0, inplace=inplace)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    torch.cuda.current_stream(dev).wait_stream(side)
    with torch.cuda.graph(graph):
        captured, norm = clip_gradients(work, 1.0, inplace=inplace)
    for k in range(4):
        for t in raw:
            t.normal_()
        raw[0] *= 10.0 ** (k - 2) / 200 if k < 2 else 1.0  # within the limit or beyond it
        for t, r in zip(work, raw):
            t.copy_(r)
        want, n = clip_gradients(raw, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(captured, want)), k


def test_more_than_32_bits_of_elements(gpu_device):
    from gsplat.gradients import clip_gradients

    dev = gpu_device
    g = torch.zeros((1 << 31) + 1003, device=dev, dtype=torch.bfloat16)
    g[0], g[-1], g[1 << 31] = 3.0, 4.0, 12.0
    out, norm = clip_gradients([g], 6.5, inplace=True)
    assert float(norm) == 13.0 and out[0] is g
    assert [float(g[0]), float(g[-1]), float(g[1 << 31])] == [1.5, 2.0, 6.0]


def test_refusals_on_the_device(gpu_device):
    from gsplat.gradients import clip_gradients

    dev = gpu_device
    flat = torch.randn(100, device=dev)
    with pytest.raises(RuntimeError, match="invalid argument"):  # one memory twice would be scaled twice
        clip_gradients([flat, flat], 1.0, inplace=True)
    with pytest.raises(RuntimeError, match="invalid argument"):
        clip_gradients([flat[:60], flat[50:]], 1.0, inplace=True)
    out, _ = clip_gradients([flat, flat], 1.0)  # read twice is fine
    assert torch.equal(out[0], out[1])
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([torch.ones(1, device=dev).expand(5)], 1.0, inplace=True)
    clip_gradients([torch.ones(1, device=dev).expand(5)], 1.0)
    with pytest.raises(TypeError):
        clip_gradients([flat.double()], 1.0)
    with pytest.raises(TypeError, match="sparse"):
        clip_gradients([flat.to_sparse()], 1.0)
    with pytest.raises(RuntimeError, match="no CPU path|different devices"):
        clip_gradients([flat, flat.cpu()], 1.0)


def test_outputs_are_ordinary_tensors(gpu_device):
    """The small ones share an allocation: nothing else about them differs."""
    import io

    from gsplat.gradients import clip_gradients, grad_norm

    dev = gpu_device
    grads = [torch.randn(7, device=dev), torch.randn(3, 5, device=dev).bfloat16(), torch.randn(4, 6, device=dev).t(), torch.empty(0, device=dev),
             torch.randn(200_000, device=dev)]
    out, norm = clip_gradients(grads, 1e-3)
    assert all(o.data_ptr() % 512 == 0 and o.stride() == g.stride() and not o.requires_grad and not o._is_view() for o, g in zip(out, grads))
    keep = [o.clone() for o in out]
    version = out[1]._version
    out[0].zero_()
    assert out[1]._version == version
    out[0] = keep[0].clone()
    assert all(torch.equal(a, b) for a, b in zip(out, keep))
    leaf = out[1].requires_grad_(True)
    (leaf.float() * 2).sum().backward()
    assert bool((leaf.grad == 2).all())
    leaf.detach().mul_(0)
    assert torch.equal(out[2], keep[2])
    buf = io.BytesIO()
    torch.save(out[2], buf)
    buf.seek(0)
    assert torch.equal(torch.load(buf, weights_only=True), keep[2])
    one, n = clip_gradients(grads[4], 1.0)  # a tensor is one gradient
    assert len(one) == 1 and one[0].shape == grads[4].shape and torch.equal(n, grad_norm(grads[4]))
    other = torch.cuda.Stream(dev)
    with torch.cuda.stream(other):  # the pool goes back to its stream's memory when the last of them is gone
        del out, leaf
        again, _ = clip_gradients(grads, 1e-3)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, keep))
