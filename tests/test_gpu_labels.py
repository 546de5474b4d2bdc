"""gsplat.losses.label_log_probs (gs_label_log_probs_fwd / _bwd) against its formula in 64 bits.

Bounds (operator_bounds.py has U = 2^-24).  With d = x - max, a term exp(d) is off by at most (3 |d| + 2) U of itself: d
and d log2 e are rounded once each, log2 e itself is off by less than U of itself, and the exponential is good to one step
(2 U).  A sum of terms that passes through c additions and scalings adds c (3 more for each scaling) U.  So, with
A = sum p |d|, A2 = sum p d^2 and c = 3 * (64 + K / 64 + 16) (a lane's share, the joins, every join a scaling):
  S relative:   e_S = (3 A + 2 + c) U            log S: e_S + 2 U |log S|
  W = sum e d:  e_W = (3 A2 + 4 A + c (A + 1)) U   entropy: e_S + e_W + e_S A + 2 U (|log S| + A)
  log p = d - log S: log S's + U (|d| + |log p|);  p: relative e_p = log p's + (2 |log p| + 2) U
  gradient: p (|c0| + |c1| (|log p| + H)) (e_p + 4 U) + p |c1| (log p's + entropy's) + (k + 2) U sum of |g| at the place,
            with c0 a sum of k + 1 terms, and one rounding.
The hardware's exponential flushes results below 2^-126 to 0: a p down there is off by up to 2^-126 (in S, whose largest
term is 1, K 2^-126 is far below U)."""
import pytest
import torch

from operator_bounds import U, assert_within, rounding

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def _reference(x, y, top, g_lp=None, g_h=None, g_top=None):
    """Values and bounds in 64 bits: dicts of (value, bound)."""
    x = x.double().cpu()
    y = y.long().cpu()
    rows, K = x.shape
    m = x.amax(1, keepdim=True)
    none = m == -INF
    d = torch.where(none, torch.full_like(x, -INF), x - m)
    e = d.exp()
    S = e.sum(1, keepdim=True)
    log_s = S.log()
    p = torch.where(none, torch.zeros_like(e), e / S)
    fin = torch.where(p > 0, d, torch.zeros_like(d))
    H = torch.where(none, torch.zeros_like(m), log_s - (p * fin).sum(1, keepdim=True))
    A, A2 = (p * fin.abs()).sum(1, keepdim=True), (p * fin * fin).sum(1, keepdim=True)
    c = 3 * (64 + K / 64 + 16)
    e_s = (3 * A + 2 + c) * U
    safe = lambda t: torch.nan_to_num(t, nan=0.0, posinf=0.0, neginf=0.0)  # noqa: E731
    b_ls = e_s + 2 * U * safe(log_s).abs()
    b_h = e_s + (3 * A2 + 4 * A + c * (A + 1)) * U + e_s * A + 2 * U * (safe(log_s).abs() + A)
    kept = (y >= 0) & (y < K)
    yy = y.clamp(0, K - 1)[:, None]
    log_p = torch.where(none, torch.full_like(x, -INF), d - log_s)
    b_log_p = b_ls + U * (safe(d).abs() + safe(log_p).abs())
    lp = torch.where(kept, log_p.gather(1, yy)[:, 0], torch.zeros(rows, dtype=torch.float64))
    res = {"log_prob": (lp, torch.where(kept, b_log_p.gather(1, yy)[:, 0], torch.zeros_like(lp))),
           "entropy": (H[:, 0], b_h[:, 0])}
    if top:
        order = torch.where(torch.isnan(x), torch.full_like(x, INF), x)
        # NaN above +inf, then the values, each by the lower index
        best = torch.stack([torch.tensor(sorted(range(K), key=lambda j, r=r: (not bool(torch.isnan(x[r, j])), -float(order[r, j]), j))[:top])
                            for r in range(rows)]) if bool(torch.isnan(x).any()) else x.sort(dim=1, descending=True, stable=True).indices[:, :top]
        t = log_p.gather(1, best)
        res["top"] = (t, b_log_p.gather(1, best))
        res["top_labels"] = best
    if g_lp is not None:
        g = torch.where(kept, g_lp.double().cpu(), torch.zeros(rows, dtype=torch.float64))[:, None]
        h = g_h.double().cpu()[:, None]
        gt = g_top.double().cpu() if top else torch.zeros(rows, 0, dtype=torch.float64)
        through, through_abs = g + gt.sum(1, keepdim=True), g.abs() + gt.abs().sum(1, keepdim=True)
        z = torch.where(p > 0, log_p, torch.zeros_like(p))
        v = p * (-through - h * torch.where(p > 0, z + H, torch.zeros_like(p)))
        size = torch.zeros_like(v)
        v.scatter_add_(1, yy, torch.where(kept[:, None], g, torch.zeros_like(g)))
        size.scatter_add_(1, yy, g.abs())
        if top:
            v.scatter_add_(1, best, gt)
            size.scatter_add_(1, best, gt.abs())
        v = torch.where(none, torch.zeros_like(v), v)
        e_p = b_log_p + (2 * safe(z).abs() + 2) * U
        weight = through_abs + h.abs() * (safe(z).abs() + safe(H))
        b = safe(p) * weight * (e_p + (6 + top) * U) + safe(p) * h.abs() * (b_log_p + b_h) + (top + 2) * U * size + 2.0 ** -126 * weight
        res["v"] = (v, b)
    return res


def _check(name, dev, x, y, top=0, grad=True, seed=0):
    from gsplat.losses import label_log_probs

    rows, K = x.shape
    g = torch.Generator().manual_seed(seed)
    g_lp, g_h, g_top = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, top, generator=g)
    xd = x.to(dev).requires_grad_(grad)
    got = label_log_probs(xd, y.to(dev), top_k=top)
    ref = _reference(x, y, top, *((g_lp, g_h, g_top) if grad else ()))
    assert got.log_prob.dtype == got.entropy.dtype == torch.float32
    assert_within(name + " log_prob", got.log_prob, *ref["log_prob"])
    assert_within(name + " entropy", got.entropy, *ref["entropy"])
    if top:
        assert torch.equal(got.top_labels.cpu(), ref["top_labels"]), name
        assert_within(name + " top", got.top_log_probs, *ref["top"])
    else:
        assert got.top_labels is None and got.top_log_probs is None
    if grad:
        outs = [got.log_prob, got.entropy] + ([got.top_log_probs] if top else [])
        ups = [g_lp.to(dev), g_h.to(dev)] + ([g_top.to(dev)] if top else [])
        (v,) = torch.autograd.grad(outs, xd, ups)
        assert v.dtype == x.dtype and v.shape == x.shape
        val, b = ref["v"]
        assert_within(name + " v", v, val, b + rounding(x.dtype, val))
    return got


def _case(rows, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, K, generator=g) * 3).to(dtype)
    return x, torch.randint(0, K, (rows,), generator=g), g


KS = [1, 2, 3, 7, 16, 19, 31, 32, 33, 63, 64, 65, 100, 127, 128, 255, 256, 257, 500, 511, 512, 513, 1000, 1023, 1024, 1025, 2047,
      2048, 2049, 4095, 4096, 4097, 5000, 8192, 9001, 16385, 32768, 50001]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", KS)
def test_every_number_of_classes(gpu_device, dtype, K):
    for rows in (1, 5, 67):
        x, y, _ = _case(rows, K, dtype, K + rows)
        _check(f"{dtype} {rows}x{K}", gpu_device, x, y, top=min(K, (rows * 3) % 9))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K", [(1, 131072), (3, 100277), (300, 40001), (700, 9000), (5000, 19), (20000, 3), (1500, 777), (4099, 64)])
def test_few_and_many_rows(gpu_device, dtype, rows, K):
    x, y, _ = _case(rows, K, dtype, rows)
    _check(f"{dtype} {rows}x{K}", gpu_device, x, y, top=3)


@pytest.mark.parametrize("K", [5, 19, 64, 65, 300, 1500, 3000, 20000])
@pytest.mark.parametrize("top", [1, 2, 5, 8, 20, 63, 64])
def test_top_of_ties(gpu_device, K, top):
    """Few distinct values: equal logits rank by the lower class, also when a row holds one value only."""
    if top > K:
        return
    g = torch.Generator().manual_seed(K + top)
    x = torch.randint(-2, 3, (9, K), generator=g).float()
    x[0] = 0.25
    x[1] = torch.where(torch.rand(K, generator=g) < 0.5, -0.0, 0.0)  # the two zeros are equal
    x[2] = torch.arange(K).float() / 100
    x[3] = -torch.arange(K).float() / 100
    x[4] = torch.finfo(torch.float32).min  # the lowest value everywhere: a uniform row
    x[5] = -INF
    y = torch.randint(0, K, (9,), generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        xx = x.to(dtype) if dtype == torch.float32 else x.clamp(min=-1e38).to(dtype)
        _check(f"ties {dtype} {K} top {top}", gpu_device, xx, y, top=top)


@pytest.mark.parametrize("K", [4, 19, 64, 65, 700, 2500, 30000])
@pytest.mark.parametrize("dtype", TYPES)
def test_masks_that_leave_little_or_nothing(gpu_device, K, dtype):
    x, y, g = _case(12, K, dtype, K)
    low = torch.finfo(dtype).min
    x[0] = -INF                                   # nothing left
    x[1] = -INF
    x[1, K - 1] = 2.0                             # one left
    x[2, : K // 2] = -INF
    x[3] = low                                    # the type's lowest value everywhere
    x[4, 1:] = low
    x[5, : K - 1] = low
    x[6] = torch.where(torch.rand(K, generator=g) < 0.9, torch.tensor(-INF), x[6].float()).to(dtype)
    x[7, 0], x[7, K - 1] = torch.finfo(dtype).max, low   # the whole range in one row
    y[8], y[9], y[10] = -1, K, -100               # void
    y[0], y[1], y[2] = 0, 0, 0                    # labels that the mask rules out
    _check(f"masked {dtype} {K}", gpu_device, x, y, top=min(K, 4))


@pytest.mark.parametrize("K", [4, 19, 64, 65, 700, 2500, 30000])
def test_nan_and_inf_stay_in_their_rows(gpu_device, K):
    from gsplat.losses import label_log_probs

    dev = gpu_device
    x, y, _ = _case(70, K, torch.float32, K)
    x[3, K // 2] = float("nan")
    x[5, 0] = INF
    x[7] = -INF
    x[7, K - 1] = float("nan")
    x[9] = float("nan")
    xd = x.to(dev).requires_grad_(True)
    got = label_log_probs(xd, y.to(dev), top_k=2)
    bad = torch.zeros(70, dtype=torch.bool)
    bad[[3, 5, 7, 9]] = True
    for t in (got.log_prob, got.entropy):
        assert torch.equal(torch.isnan(t).cpu(), bad)
    assert torch.equal(torch.isnan(got.top_log_probs).all(1).cpu(), bad)
    assert got.top_labels[3, 0] == K // 2 and got.top_labels[5, 0] == 0 and got.top_labels[7, 0] == K - 1
    assert got.top_labels[9].tolist() == [0, 1]
    (v,) = torch.autograd.grad([got.log_prob, got.entropy], xd, [torch.ones(70, device=dev)] * 2)
    assert torch.equal(torch.isnan(v).any(1).cpu(), bad)
    assert torch.equal(torch.isnan(v).all(1).cpu(), bad)


def test_rows_sum_to_zero_and_differences(gpu_device):
    """The gradient against central differences of the 64-bit formula."""
    from gsplat.losses import label_log_probs

    x, y, g = _case(4, 23, torch.float32, 5)
    y[3] = -1
    w = torch.randn(4, generator=g), torch.randn(4, generator=g), torch.randn(4, 3, generator=g)

    def f(z):
        r = _reference(z, y, 3)
        return (r["log_prob"][0] * w[0]).sum() + (r["entropy"][0] * w[1]).sum() + (r["top"][0] * w[2]).sum()

    xd = x.to(gpu_device).requires_grad_(True)
    got = label_log_probs(xd, y.to(gpu_device), 3)
    dev = gpu_device
    ((got.log_prob * w[0].to(dev)).sum() + (got.entropy * w[1].to(dev)).sum() + (got.top_log_probs * w[2].to(dev)).sum()).backward()
    z, h = x.double(), 1e-5
    for r in range(4):
        for j in range(23):
            up, down = z.clone(), z.clone()
            up[r, j] += h
            down[r, j] -= h
            assert abs(float(f(up) - f(down)) / (2 * h) - float(xd.grad[r, j])) < 2e-5
    assert float(xd.grad.double().sum(1).abs().max()) < 23 * 8 * U * 10


def test_strides_shapes_and_alignment(gpu_device):
    from gsplat.losses import label_log_probs

    dev, g = gpu_device, torch.Generator().manual_seed(2)
    render = torch.randn(2, 9, 13, 28, generator=g)
    classes = torch.randint(0, 20, (2, 9, 13), generator=g, dtype=torch.int32)
    full = render.to(dev).requires_grad_(True)
    for sl in (slice(3, 23), slice(4, 24), slice(0, 20), slice(8, 28)):  # channels of a render: a row stride of 28
        got = label_log_probs(full[..., sl], classes.to(dev), top_k=2)
        want = label_log_probs(render[..., sl].contiguous().to(dev), classes.to(dev), top_k=2)
        assert got.log_prob.shape == (2, 9, 13) and got.top_labels.shape == (2, 9, 13, 2)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        (v,) = torch.autograd.grad(got.entropy.sum() - got.log_prob.sum(), full)
        x = render[..., sl].reshape(-1, 20)
        ref = _reference(x, classes.reshape(-1), 0, -torch.ones(len(x)), torch.ones(len(x)))["v"]
        assert_within(f"slice {sl}", v[..., sl].reshape(-1, 20), ref[0], ref[1] + rounding(torch.float32, ref[0]))
        assert int((v != 0).any(0).any(0).any(0).sum()) <= 20
    t = torch.randn(20, 50, generator=g)  # classes first: copied
    got = label_log_probs(t.to(dev).t(), torch.arange(50, device=dev) % 20, 1)
    assert torch.equal(got.top_labels[:, 0].cpu(), t.t().argmax(1))
    one = label_log_probs(torch.randn(20, device=dev), torch.tensor(3, device=dev))  # no leading dimensions
    assert one.log_prob.shape == () and one.entropy.shape == ()
    wide = torch.randn(3000, 50, generator=g).to(dev)
    row = wide[:, 7].expand(6, 3000)  # rows that share memory, elements apart
    got = label_log_probs(row, torch.arange(6, device=dev), 1)
    assert bool((got.top_labels == int(wide[:, 7].argmax())).all())
    for off in range(1, 9):  # rows that start anywhere
        flat = torch.randn(5 * 3001 + 16, generator=g).bfloat16()
        a = label_log_probs(flat.to(dev)[off : off + 5 * 3001].view(5, 3001), torch.arange(5, device=dev), 4)
        b = label_log_probs(flat[off : off + 5 * 3001].view(5, 3001).clone().to(dev), torch.arange(5, device=dev), 4)
        assert torch.equal(a.top_labels, b.top_labels)
        assert float((a.log_prob - b.log_prob).abs().max()) < 1e-4


def test_empty_and_partial_gradients(gpu_device):
    from gsplat.losses import label_log_probs

    dev = gpu_device
    x = torch.zeros(0, 7, device=dev, requires_grad=True)
    got = label_log_probs(x, torch.zeros(0, dtype=torch.int64, device=dev), 2)
    assert got.log_prob.shape == (0,) and got.top_labels.shape == (0, 2)
    (got.log_prob.sum() + got.entropy.sum()).backward()
    assert x.grad.shape == (0, 7)
    xs, y, _ = _case(33, 50, torch.float32, 1)
    for pick in ("log_prob", "entropy", "top_log_probs"):
        xd = xs.to(dev).requires_grad_(True)
        got = label_log_probs(xd, y.to(dev), 4)
        (v,) = torch.autograd.grad(getattr(got, pick).sum(), xd)
        one = torch.ones(33)
        z = torch.zeros(33)
        ref = _reference(xs, y, 4, one if pick == "log_prob" else z, one if pick == "entropy" else z,
                         torch.ones(33, 4) if pick[0] == "t" else torch.zeros(33, 4))["v"]
        assert_within(pick, v, ref[0], ref[1] + rounding(torch.float32, ref[0]))


@pytest.mark.parametrize("rows,K,top", [(200, 19, 3), (3, 40000, 8), (600, 700, 5), (300, 9000, 0)])
def test_captured_replayed_and_on_another_stream(gpu_device, rows, K, top):
    from gsplat.losses import label_log_probs

    dev = gpu_device
    x = torch.randn(rows, K, device=dev).requires_grad_(True)
    y, up = torch.randint(0, K, (rows,), device=dev), torch.randn(rows, device=dev)

    def step():
        got = label_log_probs(x, y, top)
        return [t for t in got if t is not None] + [torch.autograd.grad([got.log_prob, got.entropy], x, [up, up])[0]]

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        again = step()
    for k in range(4):
        with torch.no_grad():
            x.normal_(), up.normal_(), y.random_(-1, K + 1)
        want = step()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), k
        assert all(torch.equal(a, b) for a, b in zip(again, want)), k


@pytest.mark.parametrize("rows,K", [(120_000_000, 19), (23_000, 100_003)])
def test_offsets_behind_32_bits(gpu_device, rows, K):
    from gsplat.losses import label_log_probs

    dev = gpu_device
    x = torch.zeros(rows, K, device=dev, dtype=torch.bfloat16)
    tail = torch.randn(3, K).bfloat16()
    x[-3:] = tail.to(dev)
    x.requires_grad_(True)
    y = torch.zeros(rows, dtype=torch.int32, device=dev)
    y[-3:] = torch.tensor([1, K - 1, -1])
    got = label_log_probs(x, y, 2)
    ref = _reference(tail, torch.tensor([1, K - 1, -1]), 2, torch.ones(3), torch.ones(3), torch.zeros(3, 2))
    assert_within("tail log_prob", got.log_prob[-3:], *ref["log_prob"])
    assert_within("tail entropy", got.entropy[-3:], *ref["entropy"])
    assert torch.equal(got.top_labels[-3:].cpu(), ref["top_labels"]) and got.top_labels[0].tolist() == [0, 1]
    (v,) = torch.autograd.grad([got.log_prob, got.entropy], x, [torch.ones(rows, device=dev)] * 2)
    assert_within("tail v", v[-3:], ref["v"][0], ref["v"][1] + rounding(torch.bfloat16, ref["v"][0]))


def test_refusals_on_the_device(gpu_device):
    from gsplat.losses import label_log_probs

    dev = gpu_device
    x, y = torch.randn(4, 9, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    with pytest.raises(RuntimeError, match="no CPU path"):
        label_log_probs(x, y.cpu())
    leaf = x.clone().requires_grad_(True)
    (v,) = torch.autograd.grad(label_log_probs(leaf, y).log_prob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        v.sum().backward()
    got = label_log_probs(leaf, y)
    with torch.no_grad():
        leaf.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        got.log_prob.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [300, 1000, 2047, 2048, 2049, 5003, 40001, 131072])
def test_top_where_many_are_equal(gpu_device, K, dtype):
    """Rows of mostly one value, in the places where it matters: what is above it anywhere, equal ones only at the end of
    the row or around one place, few or many above them in one thread's reach; few rows (in segments) and many."""
    from gsplat.losses import label_log_probs

    g = torch.Generator().manual_seed(K)
    rows = []
    for tie in (0.3, -0.3, -INF, 0.0):
        low = -INF if tie == -INF else tie - 1.0
        base = torch.full((K,), tie)
        rows.append(base)
        x = base.clone()  # three above
        x[torch.randint(0, K, (3,), generator=g)] = torch.tensor([1.0, 2.0, 1.0])
        rows.append(x)
        x = torch.full((K,), low)  # equal ones at the end
        x[-70:] = tie
        x[0], x[K // 2] = tie, 3.0
        rows.append(x)
        x = torch.where(torch.rand(K, generator=g) < 0.1, torch.tensor(tie), torch.tensor(low))
        rows.append(x)
        for every, count in ((256 * 4, 9), (256 * 8, 9), (64 * 4, 3), (64 * 8, 40)):  # the places of some threads' vectors
            x = base.clone()
            j = torch.arange(K)
            near = j % every < count * 4
            x[near] = torch.randint(1, 9, (int(near.sum()),), generator=g).float()
            rows.append(x)
        x = base.clone()  # more above them than any list takes
        x[::3] = torch.randint(1, 200, (len(x[::3]),), generator=g).float()
        rows.append(x)
    x = torch.stack(rows).to(dtype)
    for shift in (0, 1, 3):
        big = torch.zeros(len(rows), K + shift, dtype=dtype)
        big[:, shift:] = x
        xx = big.to(gpu_device)[:, shift:]
        y = torch.zeros(len(rows), dtype=torch.long, device=gpu_device)
        for top in (1, 5, 20, 33, 64):
            want = x.float().sort(dim=1, descending=True, stable=True).indices[:, :top]
            print(f"equal {dtype} {K} shift {shift} top {top}", flush=True)
            assert torch.equal(label_log_probs(xx, y, top_k=top).top_labels.cpu(), want)
            many = label_log_probs(xx.repeat(1100 // len(rows) + 1, 1) if shift == 0 else xx, y.repeat(1100 // len(rows) + 1) if shift == 0 else y, top_k=top)
            assert torch.equal(many.top_labels[-len(rows):].cpu(), want)
