"""Refusals of the embedding, label and gradient operators, ahead of any launch (no GPU needed)."""
import ctypes

import pytest
import torch

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3
P = 0x1000  # a non-null, 16-byte aligned dummy: never dereferenced on these paths
NULL = None


def test_embedding_entry_points_reject_bad_arguments():
    from gsplat import _backend as B

    L = B.lib()
    fwd = lambda n=4, V=3, D=2, dt=0, t=P, ts=2, ids=P, ib=8, out=P: L.gs_embedding_fwd(n, V, D, dt, t, ts, ids, ib, 1.0, out, NULL)  # noqa: E731
    for bad in (dict(n=-1), dict(V=-1), dict(D=-1), dict(dt=3), dict(dt=-1), dict(ib=2), dict(ts=-1), dict(t=NULL), dict(ids=NULL),
                dict(out=NULL), dict(t=P + 2), dict(out=P + 1), dict(ids=P + 4), dict(ids=P + 2, ib=4)):
        assert fwd(**bad) == INVALID, bad
    assert fwd(n=0) == 0 and fwd(D=0) == 0  # nothing to launch
    bwd = lambda n=4, V=3, D=2, dt=0, ids=P, ib=8, g=P, gs=2, ws=P, wb=1 << 30, out=P: L.gs_embedding_bwd(  # noqa: E731
        n, V, D, dt, ids, ib, g, gs, 1.0, ws, wb, out, NULL)
    for bad in (dict(n=-1), dict(V=-1), dict(D=-1), dict(dt=9), dict(ib=1), dict(gs=-1), dict(ids=NULL), dict(g=NULL), dict(out=NULL),
                dict(g=P + 2), dict(out=P + 2), dict(ids=P + 4), dict(n=5000, ws=NULL), dict(n=5000, ws=P + 8)):
        assert bwd(**bad) == INVALID, bad
    assert bwd(n=5000, wb=16) == WORKSPACE
    assert bwd(n=1 << 30) == UNSUPPORTED and bwd(V=1 << 31) == UNSUPPORTED
    assert bwd(V=0) == 0 and bwd(D=0) == 0
    assert L.gs_embedding_bwd_workspace_bytes(-1, 2, 3) == 0
    assert L.gs_embedding_bwd_workspace_bytes(100_000, 5000, 16) > 100_000 * 16


def test_label_entry_points_reject_bad_arguments():
    from gsplat import _backend as B

    L = B.lib()

    def fwd(rows=4, K=9, dt=0, top=2, x=P, st=9, y=P, yb=8, lp=P, ent=P, lse=P, tl=P, ti=P, ws=P, wb=1 << 30):
        return L.gs_label_log_probs_fwd(rows, K, dt, top, x, st, y, yb, ws, wb, lp, ent, lse, tl, ti, NULL)

    for bad in (dict(rows=-1), dict(K=0), dict(K=-3), dict(dt=4), dict(top=-1), dict(top=10), dict(st=-1), dict(yb=3), dict(x=NULL),
                dict(y=NULL), dict(x=P + 2), dict(y=P + 4), dict(lp=NULL), dict(ent=NULL), dict(lse=NULL), dict(tl=NULL), dict(ti=NULL)):
        assert fwd(**bad) == INVALID, bad
    assert fwd(K=100, top=65) == UNSUPPORTED
    assert fwd(rows=0) == 0

    def bwd(rows=4, K=9, dt=0, top=2, x=P, st=9, y=P, yb=8, lse=P, ent=P, ti=P, a=P, b=P, c=P, v=P):
        return L.gs_label_log_probs_bwd(rows, K, dt, top, x, st, y, yb, lse, ent, ti, a, b, c, v, NULL)

    for bad in (dict(rows=-1), dict(K=0), dict(dt=4), dict(top=10), dict(st=-1), dict(yb=3), dict(x=NULL), dict(y=NULL), dict(lse=NULL),
                dict(ent=NULL), dict(v=NULL), dict(v=P + 2), dict(ti=NULL), dict(top=0)):
        assert bwd(**bad) == INVALID, bad
    assert bwd(rows=0) == 0


def _arrays(ptrs, numels, dtypes):
    n = len(ptrs)
    return (ctypes.c_void_p * n)(*ptrs), (ctypes.c_int64 * n)(*numels), (ctypes.c_int32 * n)(*dtypes)


def test_gradient_entry_points_reject_bad_arguments():
    from gsplat import _backend as B

    L = B.lib()
    src, numel, dt = _arrays([P, 2 * P], [10, 20], [0, 1])
    dst, _, _ = _arrays([4 * P, 8 * P], [0, 0], [0, 0])
    clip = lambda n=2, s=src, d=dst, m=numel, t=dt, mx=1.0, eps=1e-6, ws=P, wb=1 << 20, out=P: L.gs_grad_clip(  # noqa: E731
        n, s, d, m, t, mx, eps, ws, wb, out, NULL)
    for bad in (dict(n=-1), dict(s=NULL), dict(d=NULL), dict(m=NULL), dict(t=NULL), dict(mx=-1.0), dict(mx=float("nan")), dict(eps=-1.0),
                dict(ws=NULL), dict(out=NULL)):
        assert clip(**bad) == INVALID, bad
    assert clip(wb=8) == WORKSPACE
    one = lambda ptr, n, t, to: clip(**dict(zip(("n", "s", "m", "t", "d"), (1, *_arrays([ptr], [n], [t]), _arrays([to], [0], [0])[0]))))  # noqa: E731
    assert one(P, 5, 7, P) == INVALID and one(P, -5, 0, P) == INVALID and one(0, 5, 0, P) == INVALID and one(P, 5, 0, 0) == INVALID
    assert one(P + 1, 5, 1, P) == INVALID and one(P, 5, 0, P + 2) == INVALID
    assert one(P, 100, 0, P + 16) == INVALID  # written onto what is still read
    two = lambda s, d: clip(**dict(zip(("s", "m", "t", "d"), (*_arrays(s, [100, 100], [0, 0]), _arrays(d, [0, 0], [0, 0])[0]))))  # noqa: E731
    assert two([P, 9 * P], [P, P]) == INVALID and two([P, P + 396], [P, P + 396]) == INVALID
    assert two([P, 9 * P], [9 * P, P]) == INVALID
    norm = lambda n=2, s=src, m=numel, t=dt, ws=P, wb=1 << 20, out=P: L.gs_grad_norm(n, s, m, t, ws, wb, out, NULL)  # noqa: E731
    for bad in (dict(n=-1), dict(s=NULL), dict(m=NULL), dict(t=NULL), dict(ws=NULL), dict(out=NULL)):
        assert norm(**bad) == INVALID, bad
    assert norm(wb=8) == WORKSPACE
    assert L.gs_grad_norm_workspace_bytes(0) > 0 and L.gs_grad_norm_workspace_bytes(100_000) >= 8 * 100_000 / 128 * 256


def test_python_entry_points_refuse():
    from gsplat.gradients import clip_grad_norm, clip_gradients, grad_norm
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    t, ids = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        embedding_lookup(t, ids)
    with pytest.raises(AssertionError):
        embedding_lookup(t[0], ids)
    for bad in (ids.to(torch.int16), ids.bool(), ids.float()):
        with pytest.raises(TypeError):
            embedding_lookup(t, bad)
    with pytest.raises(TypeError):
        embedding_lookup(t.double(), ids)
    x, y = torch.zeros(5, 9), torch.zeros(5, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        label_log_probs(x, y)
    for bad in (y[:4], y[:, None], torch.zeros(9, dtype=torch.int64)):
        with pytest.raises(AssertionError):
            label_log_probs(x, bad)
    with pytest.raises(AssertionError):
        label_log_probs(torch.zeros(5, 0), y)
    for k in (-1, 10, 65):
        with pytest.raises(ValueError, match="top_k"):
            label_log_probs(x, y, top_k=k)
    with pytest.raises(TypeError):
        label_log_probs(x.double(), y)
    with pytest.raises(TypeError):
        label_log_probs(x, y.float())
    with pytest.raises(RuntimeError, match="no CPU path"):
        clip_gradients([x], 1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        grad_norm([x])
    with pytest.raises(ValueError, match="no gradients"):
        clip_gradients([], 1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_gradients([x], bad)
    p = torch.nn.Parameter(x)
    assert float(clip_grad_norm([p], 1.0)) == 0.0  # no gradient anywhere
    with pytest.raises(TypeError, match="sparse"):
        clip_gradients([x.to_sparse()], 1.0)
