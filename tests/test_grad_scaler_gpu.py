"""Optimizers that torch.amp.GradScaler hands its scale to, on the GPU."""

import math

import pytest
import torch

from apex_amd.optimizers import FusedAdam, FusedMixedPrecisionLamb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("unscale", [False, True])
def test_fused_adam_after_unscale(unscale):
    """unscale_, clip, step: the step is that of the true gradients, bit for bit (the scale is a power of two), at an eps
    that tells their size; one that is not finite skips it."""
    g = torch.Generator().manual_seed(0)
    start = [torch.randn(s, generator=g).cuda() for s in ((3, 50), (129,), (5000,))]
    pa, pb = ([torch.nn.Parameter(w.clone()) for w in start] for _ in range(2))
    # a group: with two, the second looks at gradients that the first has unscaled
    a, b = (FusedAdam(p, lr=1e-2, eps=1e-2, bias_correction=False, capturable=True) for p in (pa, pb))
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    scaler.scale(torch.zeros((), device="cuda"))
    for step in range(3):
        for p, q in zip(pa, pb):
            q.grad = 0.02 * torch.randn(p.shape, generator=g).cuda()
            p.grad = q.grad * 1024
        if step == 1:
            pa[1].grad[7] = math.inf
        if unscale:
            scaler.unscale_(a)
            for x in (pa, pb):
                torch.nn.utils.clip_grad_norm_(x, 0.1)
        before = [p.detach().clone() for p in pa]
        scaler.step(a)
        scaler.update(1024.0)
        if step == 1:
            assert all(torch.equal(p, w) for p, w in zip(pa, before))
            continue
        b.step()
        for p, q in zip(pa, pb):
            assert torch.equal(p, q)
            for k in ("exp_avg", "exp_avg_sq"):
                assert torch.equal(a.state[p][k], b.state[q][k])


@pytest.mark.parametrize("unscale", [False, True])
def test_fused_mixed_precision_lamb_after_unscale(unscale):
    """The step is that of the true gradients at an eps that tells their size. Norms are sums of a few thousand fp32
    squares, in one order: the same but for the products with the scale's inverse."""
    g = torch.Generator().manual_seed(1)
    start = [torch.randn(s, generator=g).cuda() for s in ((3, 50), (129,), (5000,))]
    pa, pb = ([torch.nn.Parameter(w.clone()) for w in start] for _ in range(2))
    a, b = (FusedMixedPrecisionLamb(p, lr=1e-2, eps=1e-2) for p in (pa, pb))
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    scaler.scale(torch.zeros((), device="cuda"))
    for step in range(2):
        for p, q in zip(pa, pb):
            q.grad = 0.02 * torch.randn(p.shape, generator=g).cuda()
            p.grad = q.grad * 1024
        if unscale:
            scaler.unscale_(a)
        scaler.step(a)
        scaler.update(1024.0)
        b.step()
    for p, q in zip(pa, pb):
        torch.testing.assert_close(p, q, rtol=0, atol=64 * 2 ** -24)
