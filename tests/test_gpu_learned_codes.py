"""The learned-code operators together, as a training step uses them: every Gaussian takes its instance's code
(gsplat.prepass.embedding_lookup), the codes are rendered as class channels (gsplat.rendering.rasterization), the image's
class map scores them (gsplat.losses.label_log_probs), and the step's gradients are clipped
(gsplat.gradients.clip_grad_norm) before the optimizer.  Each operator is held to its formula in 64 bits on the inputs that
it met in the chain, with the bounds of operator_bounds.py."""
import pytest
import torch

import synth_scene
from operator_bounds import U, assert_within, rounding
from test_gpu_labels import _reference

pytestmark = pytest.mark.gpu


def _scene(dev, n, instances, classes, seed):
    gen = torch.Generator().manual_seed(seed)
    g = {k: v.to(dev) for k, v in synth_scene.make_gaussians(n, sh_degree=None, extent=8.0).items()}
    ids = torch.randint(0, instances, (n,), generator=gen).sort().values
    ids[torch.rand(n, generator=gen) < 0.1] = -1  # background: no instance
    codes = torch.nn.Parameter((torch.randn(instances, classes, generator=gen) * 2).to(dev))
    return g, ids.to(dev), codes


def test_a_step_with_class_channels(gpu_device):
    from gsplat.gradients import clip_grad_norm
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup
    from gsplat.rendering import rasterization

    dev, n, instances, classes, W, H = gpu_device, 3000, 90, 11, 96, 64
    g, ids, codes = _scene(dev, n, instances, classes, 3)
    means = torch.nn.Parameter(g["means"])
    vm, Ks = (t.to(dev) for t in synth_scene.make_cameras(2, W, H))
    gen = torch.Generator().manual_seed(9)
    class_map = torch.randint(-1, classes, (2, H, W), generator=gen).to(dev)
    opt = torch.optim.SGD([{"params": [codes], "lr": 0.5}, {"params": [means], "lr": 1e-3}])
    for step in range(3):
        opt.zero_grad(set_to_none=True)
        colors = embedding_lookup(codes, ids, scale=0.7)
        colors.retain_grad()
        logits, alphas, _ = rasterization(means, g["quats"], g["scales"], g["opacities"], colors, vm, Ks, W, H, near_plane=0.1,
                                          packed=False, render_mode="RGB")
        logits.retain_grad()
        got = label_log_probs(logits, class_map, top_k=2)
        loss = 0.1 * got.entropy.sum() - got.log_prob.sum()
        loss.backward()
        # lookup
        ok = ids.cpu() >= 0
        want = torch.zeros(n, classes, dtype=torch.float64)
        scale = float(torch.tensor(0.7))
        want[ok] = codes.detach().double().cpu()[ids.cpu()[ok]] * scale
        assert_within("codes", colors, want, want.abs() * U + rounding(torch.float32, want))
        # loss and its gradient on the rendered channels
        pixels = 2 * H * W
        x = logits.detach().reshape(pixels, classes)
        ref = _reference(x, class_map.reshape(-1), 2, -torch.ones(pixels), torch.full((pixels,), 0.1), torch.zeros(pixels, 2))
        assert_within("log_prob", got.log_prob.reshape(-1), *ref["log_prob"])
        assert_within("entropy", got.entropy.reshape(-1), *ref["entropy"])
        assert torch.equal(got.top_labels.reshape(-1, 2).cpu(), ref["top_labels"])
        # (0.1 in fp32 is 0.1 (1 + U) at most)
        v, b = ref["v"]
        assert_within("v_logits", logits.grad.reshape(pixels, classes), v, b * (1 + U) + v.abs() * U + rounding(torch.float32, v))
        # gradient of the codes from that of the Gaussians' colours
        up = colors.grad.double().cpu()
        row = torch.where(ok, ids.cpu(), torch.full_like(ids.cpu(), instances))
        v, size = (torch.zeros(instances + 1, classes, dtype=torch.float64).index_add_(0, row, t)[:instances] * scale for t in (up, up.abs()))
        count = torch.bincount(row, minlength=instances + 1)[:instances, None]
        assert_within("v_codes", codes.grad, v, (count + 1) * U * size + rounding(torch.float32, v))
        # clipping and the step
        raw = [p.grad.double().cpu() for p in (codes, means)]
        before = [p.detach().double().cpu() for p in (codes, means)]
        norm = torch.stack([t.square().sum() for t in raw]).sum().sqrt()
        limit = float(norm) * (0.25 if step < 2 else 4.0)
        assert_within("norm", clip_grad_norm([codes, means], limit), norm, norm * U * 1.001)
        factor = min(1.0, limit / (float(norm) + 1e-6))
        for p, t in zip((codes, means), raw):
            assert_within("clipped", p.grad, t * factor, (t * factor).abs() * 5 * U + rounding(torch.float32, t * factor))
        opt.step()
        for p, t, old, lr in zip((codes, means), raw, before, (0.5, 1e-3)):
            new = old - lr * factor * t
            assert_within("stepped", p, new, (lr * factor * t).abs() * 8 * U + new.abs() * U)


def test_a_captured_step_is_replayed(gpu_device):
    """Lookup, a linear head, loss, backward and clipping in one graph, replayed on new inputs with eager work between."""
    from gsplat.gradients import clip_gradients
    from gsplat.losses import label_log_probs
    from gsplat.prepass import embedding_lookup

    dev, n, rows, dim, classes = gpu_device, 5000, 300, 32, 19
    table = torch.randn(rows, dim, device=dev).requires_grad_(True)
    head = (torch.randn(dim, classes, device=dev) * 0.2).requires_grad_(True)
    ids, labels = torch.randint(-1, rows, (n,), device=dev), torch.randint(-1, classes, (n,), device=dev)

    def step():
        got = label_log_probs(embedding_lookup(table, ids) @ head, labels, top_k=1)
        grads = torch.autograd.grad(got.entropy.sum() * 0.1 - got.log_prob.sum(), [table, head])
        clipped, norm = clip_gradients(grads, 1.0)
        return [got.log_prob.detach(), got.top_labels, norm] + clipped

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
            table.normal_(), ids.random_(-1, rows), labels.random_(-1, classes)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            # (the library's products may choose another order of their sums under capture)
            assert torch.equal(a, b) or torch.allclose(a, b, rtol=1e-4, atol=1e-5 * float(b.abs().max())), k
