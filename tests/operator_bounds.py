"""Error bounds of the operators that the tests of embedding, labels and gradients share, from the arithmetic alone.
U = 2^-24 is half a step of fp32; a sum of c fp32 terms is off by at most c U sum|terms|; rounding to a type is off by
half a step, finfo.eps / 2, or half of its smallest subnormal."""
import torch

U = 2.0 ** -24


def rounding(dtype, ref):
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps / 2) + fi.smallest_normal * fi.eps / 2


def assert_within(name, got, ref, bound):
    """|got - ref| <= bound everywhere (bound an fp64 tensor, inflated by 1e-6 for the second order), with equal NaN and inf.
    A reference from (2 - eps / 2) 2^emax on, half a step above the type's largest value, rounds to inf in that type."""
    g, r = got.detach().double().cpu(), ref.detach().double().cpu()
    fi = torch.finfo(got.dtype)
    r = torch.where(r.abs() >= fi.max * (1 + fi.eps / 4), r.sign() * float("inf"), r)
    b = torch.as_tensor(bound, dtype=torch.float64).detach().cpu().expand_as(r)
    assert g.shape == r.shape, (name, g.shape, r.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(r)), f"{name}: NaN in other places"
    inf = torch.isinf(r) | torch.isinf(g)
    assert torch.equal(g[inf], r[inf]), f"{name}: infinities differ"
    ok = ~inf & ~torch.isnan(r)
    err, b = (g - r).abs()[ok], b[ok] * (1 + 1e-6)
    bad = err > b
    worst = float((err / b.clamp(min=1e-300)).max()) if err.numel() else 0.0
    print(f"[bound] {name}: n={err.numel()} worst error {worst:.3f} of the bound")
    assert not bool(bad.any()), f"{name}: {int(bad.sum())} of {err.numel()} outside the bound, worst {worst:.3f} times"
