"""Token losses on the GPU against 64 bits, at the sizes that choose the blocks: long sequences (1024 threads each), rows
of every block size, and every number of packs that the policy gradient holds in registers. The bounds are those of
test_token_loss_gpu."""

import pytest
import torch

import token_loss_oracle as oracle
from apex_amd.contrib.xentropy import policy_loss, preference_loss, sequence_log_probs, token_log_probs
from test_token_loss_gpu import DTYPES, U, grad_of, make, near, policy_bounds, sum_bound

pytestmark = pytest.mark.gpu

VOCAB = 65


def long(length, packed, dtype):
    """Four sequences of over 512 rows in the mean: padded ones, one of them masked whole; or packed ones with rows in
    front and behind, one empty and one of twice the length."""
    if not packed:
        x, y, g = make((4, length), VOCAB, dtype)
        y[1] = -100
        y[3, length // 3:] = -100
        return x, y, g, None, None
    cu = [3, 3 + 2 * length, 3 + 2 * length, 4 + 3 * length, 2 + 4 * length]
    x, y, g = make((4 * length + 5,), VOCAB, dtype)
    return x, y, g, cu, torch.tensor(cu, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("length", [513, 1500])
@pytest.mark.parametrize("average", [False, True])
def test_long_sequence_log_probs(length, packed, average):
    x, y, g, cu, cug = long(length, packed, torch.float32)
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want = oracle.sums(oracle.log_probs(x64, y), y, cu=cu, average=average)
    got = sequence_log_probs(xg, y.cuda(), cug, average=average)
    near(got, want, sum_bound(x, y, cu, average) + U * want.detach().abs())
    w = torch.randn(4, generator=g)
    lp = torch.zeros(y.numel(), dtype=torch.float64, requires_grad=True)
    coef = torch.autograd.grad(oracle.sums(lp, y, cu=cu, average=average), lp, w.double())[0].view(y.shape)
    near(grad_of(got, xg, w), torch.autograd.grad(want, x64, w.double())[0], oracle.grad_bound(x, y, coef, torch.float32))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("length", [513, 1500])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_preference_loss(length, packed, average, dtype):
    x, y, g, cu, cug = long(length, packed, dtype)
    beta, scale = 0.25, 1024.0
    ref = (oracle.sums(oracle.log_probs(x.double(), y), y, cu=cu, average=average) + torch.randn(4, generator=g)).float()
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, gain = oracle.preference(x64, y, ref, beta, 0.1, "sigmoid", average, cu)
    loss, chosen, rejected = preference_loss(xg, y.cuda(), ref.cuda(), beta, 0.1, "sigmoid", average, cug)
    off = sum_bound(x, y, cu, average)
    near(torch.cat([chosen, rejected]), gain, beta * off + 2 * U * gain.abs())
    off = off[:2] + off[2:]  # of a pair's difference; the slope is under beta, and its own slope under beta^2 / 4
    near(loss, want, (beta * off).mean() + 2 * U * want.detach().abs())
    lp = torch.zeros(y.numel(), dtype=torch.float64, requires_grad=True)
    sign = torch.tensor([1.0, 1.0, -1.0, -1.0]).double() / 2 * scale
    each = oracle.sums(lp, y, cu=cu, average=average)
    coef = torch.autograd.grad(each, lp, sign * beta, retain_graph=True)[0].view(y.shape)
    wander = torch.autograd.grad(each, lp, sign * (beta ** 2 / 4 * off).repeat(2))[0].view(y.shape)
    dx = grad_of(loss, xg, torch.tensor(scale))
    near(dx, torch.autograd.grad(want, x64)[0] * scale, oracle.grad_bound(x, y, coef, dtype) + 2 * wander.abs().unsqueeze(-1))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("length", [513, 1500])
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
@pytest.mark.parametrize("scale", [None, 512.0])
def test_long_policy_loss(length, packed, reduction, scale):
    dtype, kl = torch.float32, 0.05
    x, y, g, cu, cug = long(length, packed, dtype)
    lp = oracle.log_probs(x.double(), y).float()
    move = 0.3 * torch.randn(y.shape, generator=g)
    for border in (0.8, 1.2):  # fp32 cannot tell a ratio's side within its own error of a border
        move = torch.where((move + torch.tensor(border).log()).abs() < 1e-3, 0.0, move)
    old, ref = lp + move, lp + 0.5 * torch.randn(y.shape, generator=g)
    adv = torch.randn(4, generator=g)
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, _ = oracle.policy(x64, y, old, adv, ref, kl=kl, reduction=reduction, cu=cu)
    loss, got = policy_loss(xg, y.cuda(), old.cuda(), adv.cuda(), ref.cuda(), kl_coef=kl, reduction=reduction, cu_seqlens=cug, grad_scale=scale)
    near(got, lp.double(), oracle.lp_bound(x, y) + U * lp.double().abs())
    size, off = policy_bounds(x, y, old, ref, adv, kl, 1.0, cu)
    inside = torch.zeros(y.numel(), dtype=torch.bool)
    for a, e in oracle.spans(y, cu):
        inside[a:e] = True
    inside = inside.view(y.shape) & (y != -100)
    ones = torch.zeros(y.numel(), dtype=torch.float64, requires_grad=True)
    weight = {"token": lambda: inside / inside.sum(), "sum": lambda: inside.double(),
              "sequence": lambda: torch.autograd.grad(oracle.sums(ones, y, cu=cu, average=True).mean(), ones)[0].view(y.shape) * inside}[reduction]()
    near(loss, want, (weight * (off + 4 * U * size)).sum() + 2 * U * want.detach().abs())
    weight = weight * 512.0
    bound = oracle.grad_bound(x, y, weight * size, dtype) + (weight * off).abs().unsqueeze(-1)
    near(grad_of(loss, xg, torch.tensor(512.0)), torch.autograd.grad(want, x64)[0] * 512.0, bound)


# packs of 16 bytes a row: 64 lanes up to 512; then 512 for up to 512 rows, 256 for up to 1023, 128 for more up to 1536
@pytest.mark.parametrize("packs", [90, 600, 1000, 1400, 2000])
@pytest.mark.parametrize("rows", [9, 700, 1031])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_each_block(packs, rows, dtype):
    x, y, g = make((rows,), packs * (16 // dtype.itemsize) + 1, dtype, ignored=0.9 if rows > 9 else 0.1)
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, got = oracle.log_probs(x64, y), token_log_probs(xg, y.cuda())
    near(got, want, oracle.lp_bound(x, y))
    w = torch.randn(y.shape, generator=g)
    on = y != -100
    dx, wanted = grad_of(got, xg, w), torch.autograd.grad(want, x64, w.double())[0]
    near(dx[on.cuda()], wanted[on], oracle.grad_bound(x[on], y[on], w[on], dtype))
    assert not dx[~on.cuda()].any()


# one size within each of the register tiers: 64, 256, 512 and 1024 lanes of 2 to 16 packs
@pytest.mark.parametrize("packs", [100, 200, 300, 450, 800, 1300, 1800, 2300, 2800, 3300, 3900, 4600, 5600, 6600, 7700, 9000, 11000, 13000, 15000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_at_once_in_each_tier(packs, dtype):
    x, y, _ = make((2, 2), packs * (16 // dtype.itemsize) + 3, dtype, ignored=0)
    lp = oracle.log_probs(x.double(), y).float()
    old, adv = lp + 0.05, torch.tensor([1.5, -0.5])
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, _ = oracle.policy(x64, y, old, adv)
    loss, got = policy_loss(xg, y.cuda(), old.cuda(), adv.cuda(), grad_scale=64.0)
    near(got, lp.double(), oracle.lp_bound(x, y) + U * lp.double().abs())
    size, off = policy_bounds(x, y, old, None, adv, 0.0, 1.0, None)
    near(loss, want, ((off + 4 * U * size) / 4).sum() + 2 * U * want.detach().abs())
    dx = grad_of(loss, xg, torch.tensor(64.0))
    bound = oracle.grad_bound(x, y, size * 16, dtype) + (off * 16).unsqueeze(-1)
    near(dx, torch.autograd.grad(want, x64)[0] * 64, bound)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_sum_keeps_what_is_far_under_its_largest_term(dtype):
    """One term of 1 and 131071 of 2^-27, which fp32 loses where it adds packs of them to the 1: some 2e-6 in each row's
    log-probability. The small terms are off by 8 half steps of fp32 of their sum (1e-3) together. The pack that holds
    the 1 is added in fp32: three sums of a little over 1, each off by at most half a step of it, 2^-24."""
    x = torch.full((140, 131072), -18.75).to(dtype)
    x[:, 0] = 0
    y = torch.zeros(140, 1, dtype=torch.long)
    lp = -torch.logsumexp(x[0].double(), -1)
    xg = x.cuda().view(140, 1, -1).requires_grad_(True)
    ref = lp.float().expand(140).contiguous()
    _, chosen, rejected = preference_loss(xg, y.cuda(), ref.cuda(), beta=1.0)
    want = lp - ref.double()
    near(torch.cat([chosen, rejected]), want, 3 * U + 8 * U * lp.abs() + U * want.abs())
    # one in 32 bits takes the sum rounded once more, and its log2
    for got in (token_log_probs(xg, y.cuda()), policy_loss(xg, y.cuda(), None, torch.ones(140, device="cuda"), grad_scale=1.0)[1]):
        near(got, lp.expand(140, 1), torch.tensor(3 * U + 4 * U))
