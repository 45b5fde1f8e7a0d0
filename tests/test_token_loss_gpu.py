"""Token losses on the GPU against 64 bits: vocabularies of every remainder, layouts, masks, both ways of the policy
gradient, streams and graphs. The bounds count half steps of fp32 and one rounding of the result (token_loss_oracle)."""

import math

import pytest
import torch

import token_loss_oracle as oracle
from apex_amd.contrib.xentropy import policy_loss, preference_loss, sequence_log_probs, token_log_probs

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
U = oracle.U


def make(lead, vocab, dtype, seed=0, ignored=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*lead, vocab, generator=g) * 2.5).to(dtype)
    y = torch.randint(0, vocab, lead, generator=g)
    y[torch.rand(lead, generator=g) < ignored] = -100
    return x, y, g


def near(got, want, bound):
    got, want = got.detach().cpu().double(), want.detach().double()
    assert got.shape == want.shape
    both = torch.isnan(got) & torch.isnan(want) | (got == want)
    off = torch.where(both, 0.0, (got - want).abs() - bound)
    assert not torch.isnan(off).any() and (off <= 0).all(), f"{(off > 0).sum()} of {off.numel()} out of bounds, by {off.max():.3g}"


def grad_of(out, x, w):
    return torch.autograd.grad(out, x, w.to(x.device) if torch.is_tensor(w) else w)[0]


# 1 to 17: under and around a pack; 2048, 2051: a block's pass; 40000 and up: rows that many lanes or registers share
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 17, 255, 2048, 2051, 32000, 40001, 70003, 131077])
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_log_probs(vocab, dtype):
    x, y, g = make((2, 4), vocab, dtype)
    t = 0.7
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, got = oracle.log_probs(x64, y, temperature=t), token_log_probs(xg, y.cuda(), temperature=t)
    assert got.dtype == torch.float32
    near(got, want, oracle.lp_bound(x, y, temperature=t))
    w = torch.randn(y.shape, generator=g)
    dx = grad_of(got, xg, w)
    assert dx.dtype == dtype
    near(dx, torch.autograd.grad(want, x64, w.double())[0], oracle.grad_bound(x, y, w, dtype, temperature=t))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", ["swapped", "shorter", "narrow", "offset", "spread", "expanded", "four", "one", "flat"])
def test_layouts(layout, dtype):
    """Rows that lie apart, at odd addresses, over each other, or with spaces inside."""
    V = 517
    base, _, g = make((3, 4), V + 3, dtype)
    view = {
        "swapped": lambda b: b[..., :V].transpose(0, 1),
        "shorter": lambda b: b[:, :-1, :V],
        "narrow": lambda b: b[..., :V],
        "offset": lambda b: b[..., 3:],
        "spread": lambda b: b[..., :V - 1:2],
        "expanded": lambda b: b[:, :1, :V].expand(3, 5, V),
        "four": lambda b: b[..., :V].unsqueeze(1).expand(3, 2, 4, V).transpose(1, 2),
        "one": lambda b: b[1, 2, :V],
        "flat": lambda b: b.reshape(12, V + 3)[1:11:3, 1:],
    }[layout]
    x = view(base)
    y = torch.randint(0, x.shape[-1], x.shape[:-1], generator=g)
    w = torch.randn(y.shape, generator=g)
    b64, bg = base.double().requires_grad_(True), base.cuda().requires_grad_(True)
    want, got = oracle.log_probs(view(b64), y), token_log_probs(view(bg), y.cuda())
    near(got, want, oracle.lp_bound(x, y))
    bound = torch.zeros_like(base, dtype=torch.float64)
    each = oracle.grad_bound(x, y, w, dtype)
    # an element that is met several times sums several gradients, each rounded, and the sums are rounded again
    where = view(torch.arange(base.numel()).view(base.shape)).reshape(-1)
    bound.view(-1).index_add_(0, where, each.reshape(-1))
    size = torch.zeros_like(bound)
    size.view(-1).index_add_(0, where, (w.abs().double().unsqueeze(-1).expand(each.shape)).reshape(-1))
    times = torch.bincount(where, minlength=base.numel()).max().item()
    if times > 1:
        bound = bound + size * (times - 1) * torch.finfo(dtype).eps / 2
    near(grad_of(got, bg, w), torch.autograd.grad(want, b64, w.double())[0], bound)


def test_int32_labels_and_no_rows():
    x, y, _ = make((3, 4), 100, torch.float32)
    a, b = token_log_probs(x.cuda(), y.cuda()), token_log_probs(x.cuda(), y.int().cuda())
    assert torch.equal(a, b)
    x = torch.empty(3, 0, 100, device="cuda", requires_grad=True)
    lp = token_log_probs(x, torch.empty(3, 0, dtype=torch.long, device="cuda"))
    assert lp.shape == (3, 0)
    lp.sum().backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("vocab", [19, 5000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_edges(vocab, dtype):
    low = torch.finfo(dtype).min
    x, y, _ = make((1, 9), vocab, dtype, ignored=0)
    x[0, 0, 1:] = -math.inf          # one token left, and it is the label
    y[0, 0] = 0
    x[0, 1, :-1] = low               # the type's lowest value as a mask
    y[0, 1] = vocab - 1
    x[0, 2] = -math.inf              # nothing left
    x[0, 3, 2] = math.inf
    x[0, 4, 2] = math.nan
    x[0, 5, 1] = -math.inf           # the label itself is masked
    y[0, 5] = 1
    x[0, 6] = 7.0                    # all the same
    x[0, 7], y[0, 7] = math.nan, -100
    x[0, 8], y[0, 8] = math.inf, -100
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, got = oracle.log_probs(x64, y), token_log_probs(xg, y.cuda())
    bound = oracle.lp_bound(x, y)
    bound[0, 1] = oracle.lp_bound(x[:, 6:7], y[:, 6:7])[0, 0]  # the lowest values are no part of the sum
    near(got, want, bound)
    v = got.detach()
    assert math.isnan(v[0, 2]) and math.isnan(v[0, 4]) and v[0, 5] == -math.inf and v[0, 7] == 0 and v[0, 8] == 0
    assert got[0, 0] == 0 and got[0, 1].abs() < 1e-3
    dx = grad_of(got, xg, torch.ones_like(got))
    assert (dx[0, 7:] == 0).all()
    assert torch.isfinite(dx[0, [0, 1, 5, 6]]).all() and torch.isnan(dx[0, 2]).all()
    assert (dx[0, 0] == 0).all()


def test_labels_out_of_range_are_nan():
    x, y, _ = make((2, 3), 50, torch.float32, ignored=0)
    y[0, 1], y[1, 2] = 50, -7
    x = x.cuda().requires_grad_(True)
    lp = token_log_probs(x, y.cuda())
    dx = grad_of(lp, x, torch.ones_like(lp))
    bad = (y < 0) | (y >= 50)
    assert torch.equal(torch.isnan(lp).cpu(), bad)
    assert torch.equal(torch.isnan(dx).all(-1).cpu(), bad) and torch.isfinite(dx[~bad.cuda()]).all()


def test_an_ignore_index_of_the_vocabulary():
    x, y, _ = make((2, 30), 5, torch.float32, ignored=0)
    lp = token_log_probs(x.cuda(), y.cuda(), ignore_index=2).cpu()
    assert (lp[y == 2] == 0).all() and (lp[y != 2] < 0).all()


# a token before the first sequence, an empty one, one that is ignored whole, and tokens behind the last
CU = [1, 40, 40, 43, 300, 301, 340]
ROWS = 350


def layout_of(packed, vocab, dtype):
    x, y, g = make((ROWS,) if packed else (6, 50), vocab, dtype)
    if packed:
        y[40:43] = -100
    else:
        y[2] = -100
    return x, y, g, CU if packed else None, torch.tensor(CU, dtype=torch.int32, device="cuda") if packed else None


def sum_bound(x, y, cu, average):
    on = (y != -100).view(-1)
    b = oracle.lp_bound(x, y).view(-1)
    out = [b[s:e].sum() / (max(1, int(on[s:e].sum())) if average else 1) for s, e in oracle.spans(y, cu)]
    return torch.stack(out)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sequence_log_probs(dtype, average, packed):
    x, y, g, cu, cug = layout_of(packed, 203, dtype)
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want = oracle.sums(oracle.log_probs(x64, y), y, cu=cu, average=average)
    got = sequence_log_probs(xg, y.cuda(), cug, average=average)
    near(got, want, sum_bound(x, y, cu, average) + U * want.detach().abs())
    w = torch.randn(6, generator=g)
    lp = torch.zeros(y.numel(), dtype=torch.float64, requires_grad=True)
    coef = torch.autograd.grad(oracle.sums(lp, y, cu=cu, average=average), lp, w.double())[0].view(y.shape)
    near(grad_of(got, xg, w), torch.autograd.grad(want, x64, w.double())[0], oracle.grad_bound(x, y, coef, dtype))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("kind,smoothing,average", [("sigmoid", 0.0, False), ("sigmoid", 0.3, True), ("ipo", 0.0, True), ("hinge", 0.0, False)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_preference_loss(dtype, kind, smoothing, average, packed):
    x, y, g, cu, cug = layout_of(packed, 203, dtype)
    lp = oracle.log_probs(x.double(), y)
    ref = (oracle.sums(lp, y, cu=cu, average=average) + torch.randn(6, generator=g)).float()
    beta = 0.25
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, gain = oracle.preference(x64, y, ref, beta, smoothing, kind, average, cu)
    loss, chosen, rejected = preference_loss(xg, y.cuda(), ref.cuda(), beta, smoothing, kind, average, cug)
    assert loss.shape == () and not chosen.requires_grad
    off = sum_bound(x, y, cu, average)  # of each sequence's sum
    near(torch.cat([chosen, rejected]), gain, beta * off + 2 * U * gain.abs())
    d = (gain[:3] - gain[3:]) / beta
    # a pair's d is off by its two sums' bounds; the loss by its slope times that, the slope by its own slope
    off = off[:3] + off[3:]
    slope, bend = {"sigmoid": (beta, beta ** 2 / 4), "hinge": (beta, 0.0), "ipo": (2 * (d - 0.5 / beta).abs() + off, 2.0)}[kind]
    near(loss, want, (slope * off).mean() + 2 * U * want.detach().abs())
    scale = 1024.0
    dx = grad_of(loss, xg, torch.tensor(scale))
    flat = torch.zeros(y.numel(), dtype=torch.float64, requires_grad=True)
    s = torch.cat([torch.ones(3), -torch.ones(3)]).double() / 3
    per = torch.cat([slope * torch.ones(3), slope * torch.ones(3)]).double() if not torch.is_tensor(slope) else torch.cat([slope, slope])
    coef = torch.autograd.grad(oracle.sums(flat, y, cu=cu, average=average), flat, s * per)[0].view(y.shape) * scale
    wander = torch.autograd.grad(oracle.sums(flat, y, cu=cu, average=average), flat, s * torch.cat([bend * off, bend * off]))[0].view(y.shape) * scale
    bound = oracle.grad_bound(x, y, coef, dtype) + 2 * wander.abs().unsqueeze(-1)
    near(dx, torch.autograd.grad(want, x64)[0] * scale, bound)


@pytest.mark.parametrize("shift", [-1e5, -3e3, 3e3, 1e5])
@pytest.mark.parametrize("kind", ["sigmoid", "hinge"])
def test_preference_far_out(kind, shift):
    """Differences whose exponentials overflow or vanish."""
    x, y, _ = make((2, 9), 33, torch.float32)
    ref = torch.tensor([0.0, shift])
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, _ = oracle.preference(x64, y, ref, 0.1, 0.0, kind)
    loss, _, _ = preference_loss(xg, y.cuda(), ref.cuda(), 0.1, 0.0, kind)
    near(loss, want, 0.1 * sum_bound(x, y, None, False).sum() + 2 * U * want.detach().abs())
    dx, want = grad_of(loss, xg, torch.tensor(1.0)), torch.autograd.grad(want, x64)[0]
    near(dx, want, oracle.grad_bound(x, y, torch.full(y.shape, 0.1), torch.float32))


@pytest.mark.parametrize("kind", ["sigmoid", "hinge"])
def test_a_rejected_answer_that_cannot_be(kind):
    """A rejected token of probability 0: the pair is as right as can be, and asks for nothing."""
    x = torch.zeros(2, 3, 5, device="cuda")
    x[1, 1, 4] = -math.inf
    y = torch.tensor([[0, 1, 2], [3, 4, 0]], device="cuda")
    x.requires_grad_(True)
    loss, _, rejected = preference_loss(x, y, torch.zeros(2, device="cuda"), loss_type=kind)
    assert loss == 0 and rejected[0] == -math.inf
    loss.backward()
    assert (x.grad == 0).all()


def test_nothing_is_labelled():
    """Whole batches of padding: losses of 0 (or of the references alone), gradients of 0."""
    x = torch.full((4, 3, 9), math.nan, device="cuda", requires_grad=True)
    y = torch.full((4, 3), -100, device="cuda")
    adv = torch.ones(4, device="cuda")
    for reduction in ("token", "sequence", "sum"):
        for scale in (None, 1.0):
            loss, lp = policy_loss(x, y, None, adv, reduction=reduction, grad_scale=scale)
            assert loss == 0 and (lp == 0).all()
            assert (grad_of(loss, x, torch.tensor(1.0)) == 0).all()
    loss, chosen, _ = preference_loss(x, y, adv, average=True)
    assert abs(float(loss.detach()) - math.log(2)) < 1e-6 and (chosen == -0.1 * adv[:2]).all()
    assert (grad_of(loss, x, torch.tensor(1.0)) == 0).all()
    assert (sequence_log_probs(x, y, average=True) == 0).all()


def test_one_token():
    x, y, _ = make((1, 1), 32000, torch.bfloat16, ignored=0)
    got = token_log_probs(x.cuda(), y.cuda())
    near(got, oracle.log_probs(x.double(), y), oracle.lp_bound(x, y))
    assert torch.equal(sequence_log_probs(x.cuda(), y.cuda()), got.view(1))
    flat = policy_loss(x.cuda().view(1, 32000), y.cuda().view(1), None, torch.ones(1, device="cuda"))[0]
    assert flat.item() == -1.0


def test_many_rows_of_a_small_vocabulary():
    """More rows than a grid has blocks along one side, more sequences than a block has threads."""
    x, y, g = make((70000,), 6, torch.float32)
    cu = torch.arange(0, 70001, 7, dtype=torch.int32)
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    lp = oracle.log_probs(x64, y)
    got = sequence_log_probs(xg, y.cuda(), cu.cuda())
    near(got, lp.view(-1, 7).sum(1), oracle.lp_bound(x, y).view(-1, 7).sum(1) + U * 100)
    near(grad_of(got, xg, torch.ones(10000)), torch.autograd.grad(lp.sum(), x64)[0], oracle.grad_bound(x, y, torch.ones(70000), torch.float32))
    adv = torch.randn(10000, generator=g)
    want, _ = oracle.policy(x.double(), y, None, adv, reduction="sequence", cu=cu.tolist())
    for scale in (None, 1.0):
        loss, _ = policy_loss(xg, y.cuda(), None, adv.cuda(), reduction="sequence", cu_seqlens=cu.cuda(), grad_scale=scale)
        # 10^4 means of -A, each rounded a few times; their sum in 64 bits
        near(loss, want, 4 * U * adv.abs().mean().double())


def policy_case(packed, dtype, vocab, by_row, kl, on_policy, temperature, seed=0):
    x, y, g, cu, cug = layout_of(packed, vocab, dtype)
    lp = oracle.log_probs(x.double(), y, temperature=temperature).float()
    move = 0.3 * torch.randn(y.shape, generator=g)
    for border in (0.8, 1.3):  # fp32 cannot tell a ratio's side within its own error of a border
        move = torch.where((move + math.log(border)).abs() < 1e-3, 0.0, move)
    old = None if on_policy else torch.where(y == -100, math.nan, lp + move)  # ignored tokens may hold anything
    ref = torch.where(y == -100, math.inf, lp + 0.5 * torch.randn(y.shape, generator=g)) if kl else None
    adv = torch.randn(y.shape if by_row else (6,), generator=g)
    return x, y, cu, cug, old, ref, adv, g


def policy_bounds(x, y, old, ref, adv, kl, t, cu):
    """Of each token's loss, the size of its slope, and how far the slope may be: dlp moves a ratio by ratio dlp, and KL's slope by exp(d) dlp."""
    lp = oracle.log_probs(x.double(), y, temperature=t)
    on = y != -100
    b = oracle.lp_bound(x, y, temperature=t) + 4 * U * lp.abs()
    owner = torch.zeros(y.numel(), dtype=torch.long)
    for s, (a, e) in enumerate(oracle.spans(y, cu)):
        owner[a:e] = s
    A = (adv if adv.shape == y.shape else adv[owner].view(y.shape)).double().abs()
    ratio = torch.ones_like(lp) if old is None else torch.where(on, torch.exp(lp - old.double()), 1.0)
    grown = torch.where(on, torch.exp(ref.double() - lp), 0.0) if ref is not None else torch.zeros_like(lp)
    size = ratio * A + kl * (grown + 1)
    off = torch.where(on, (ratio * A + kl * (grown + 1)) * (2 * b + 8 * U), 0.0)
    return torch.where(on, size, 0.0), off


@pytest.mark.parametrize("packed,by_row,kl,on_policy", [(False, False, 0.1, False), (False, True, 0.0, True), (True, False, 0.05, True), (True, True, 0.1, False)])
@pytest.mark.parametrize("reduction", ["token", "sequence", "sum", "none"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_loss(dtype, reduction, packed, by_row, kl, on_policy):
    t = 0.8
    x, y, cu, cug, old, ref, adv, g = policy_case(packed, dtype, 203, by_row, kl, on_policy, t)
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, lp = oracle.policy(x64, y, old, adv, ref, high=0.3, kl=kl, temperature=t, reduction=reduction, cu=cu)
    args = dict(clip_eps_high=0.3, kl_coef=kl, temperature=t, reduction=reduction, cu_seqlens=cug)
    given = [None if v is None else v.cuda() for v in (old, adv, ref)]
    loss, got = policy_loss(xg, y.cuda(), given[0], given[1], given[2], **args)
    near(got, lp, oracle.lp_bound(x, y, temperature=t))
    size, off = policy_bounds(x, y, old, ref, adv, kl, t, cu)
    # each token's weight in the loss
    ones = torch.zeros(y.numel(), dtype=torch.float64, requires_grad=True)
    inside = torch.zeros(y.numel(), dtype=torch.bool)
    for a, e in oracle.spans(y, cu):
        inside[a:e] = True
    inside = inside.view(y.shape) & (y != -100)
    count = inside.sum()
    weight = {"token": lambda: inside / count, "sum": lambda: inside.double(), "none": lambda: inside.double(),
              "sequence": lambda: torch.autograd.grad(oracle.sums(ones, y, cu=cu, average=True).mean(), ones)[0].view(y.shape) * inside}[reduction]()
    if reduction == "none":
        near(loss, want, off + 4 * U * size)
        w = torch.randn(y.shape, generator=g)
    else:
        near(loss, want, (weight * (off + 4 * U * size)).sum() + 2 * U * want.detach().abs())
        w = torch.tensor(512.0)
    dx = grad_of(loss, xg, w)
    want = torch.autograd.grad(want, x64, w.double())[0]
    weight = weight * w.double()
    bound = oracle.grad_bound(x, y, weight * size, dtype, temperature=t) + ((weight * off).abs() / t).unsqueeze(-1)
    near(dx, want, bound)
    if reduction == "none":
        return
    # the gradient of the forward pass, for a scale as a number and as a value on the device
    for scale in (512.0, torch.tensor(512.0, device="cuda")):
        loss1, got1 = policy_loss(xg, y.cuda(), given[0], given[1], given[2], grad_scale=scale, **args)
        near(got1, lp, oracle.lp_bound(x, y, temperature=t))
        near(loss1, loss.detach().cpu(), (weight / 512 * (2 * off + 8 * U * size)).sum() + 2 * U * loss.detach().cpu().double().abs())
        near(grad_of(loss1, xg, w), want, bound)


@pytest.mark.parametrize("vocab", [5, 8, 4099, 32768, 32769, 65537, 131072, 131079])
@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_at_once(dtype, vocab):
    """Rows of every size that a block's registers hold, and longer ones."""
    x, y, g = make((2, 3), vocab, dtype, ignored=0)
    y[1, 2] = -100
    lp = oracle.log_probs(x.double(), y).float()
    old, adv = lp + 0.05, torch.tensor([1.5, -0.5])
    x64, xg = x.double().requires_grad_(True), x.cuda().requires_grad_(True)
    want, _ = oracle.policy(x64, y, old, adv)
    loss, got = policy_loss(xg, y.cuda(), old.cuda(), adv.cuda(), grad_scale=64.0)
    near(got, lp.double(), oracle.lp_bound(x, y) + U * lp.double().abs())
    size, off = policy_bounds(x, y, old, None, adv, 0.0, 1.0, None)
    near(loss, want, ((off + 4 * U * size) / 5).sum() + 2 * U * want.detach().abs())
    dx = grad_of(loss, xg, torch.tensor(64.0))
    bound = oracle.grad_bound(x, y, size * 64 / 5, dtype) + (off * 64 / 5).unsqueeze(-1)
    near(dx, torch.autograd.grad(want, x64)[0] * 64, bound)


def test_policy_at_once_with_another_gradient_and_twice():
    x, y, g = make((2, 5), 300, torch.bfloat16, ignored=0)
    adv = torch.tensor([1.0, -2.0], device="cuda")
    xg = x.cuda().requires_grad_(True)
    loss, _ = policy_loss(xg, y.cuda(), None, adv, grad_scale=4.0)
    dx = torch.autograd.grad(loss * 3.0, xg, retain_graph=True)[0]
    want = torch.autograd.grad(policy_loss(xg, y.cuda(), None, adv)[0] * 3.0, xg)[0]
    # one rounding more than the direct gradient, and one of the quotient
    near(dx, want.cpu().double(), want.cpu().double().abs() * (2 * torch.finfo(torch.bfloat16).eps / 2 + 4 * U) * 1.01)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(loss * 3.0, xg)
    with torch.no_grad():
        plain, _ = policy_loss(xg, y.cuda(), None, adv, grad_scale=4.0)
    assert torch.equal(plain, loss.detach())


@pytest.mark.parametrize("cu", [[-5, 3, 2, 900], [400, 500, 600, 700], [0, 0, 0, 0]])
def test_cu_seqlens_that_do_not_fit_stay_inside(cu):
    x, y, _ = make((ROWS,), 40, torch.float32, ignored=0)
    c = torch.tensor(cu, dtype=torch.int32, device="cuda")
    xg = x.cuda().requires_grad_(True)
    got = sequence_log_probs(xg, y.cuda(), c)
    got.sum().backward()
    lp = oracle.log_probs(x.double(), y)
    want = []
    for a, b in zip(cu, cu[1:]):
        a = min(max(a, 0), ROWS)
        want.append(lp[a:min(max(b, a), ROWS)].sum())
    near(got, torch.stack(want), oracle.lp_bound(x, y).sum() + U * 2000)


def test_another_stream_and_the_same_results_again():
    x, y, _ = make((6, 50), 5003, torch.bfloat16)
    ref = torch.full((6,), -300.0).cuda()
    xg, yg = x.cuda().requires_grad_(True), y.cuda()

    def run():
        loss, a, b = preference_loss(xg, yg, ref, 0.01)
        return [loss.detach(), a, b, grad_of(loss, xg, torch.tensor(1.0))]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.synchronize()
    for _ in range(3):
        for a, b in zip(first, again):
            assert torch.equal(a, b)
        again = run()


@pytest.mark.parametrize("which", ["tokens", "pairs", "policy", "at once"])
def test_captured_and_replayed(which):
    """Three replays on new values, with eager work between, each equal to the eager result."""
    xs = [make((4, 30), 1003, torch.bfloat16, seed=s)[0].cuda() for s in range(3)]
    y = make((4, 30), 1003, torch.bfloat16)[1].cuda()
    ref, adv = torch.full((4,), -100.0).cuda(), torch.randn(4).cuda()
    scale = torch.ones((), device="cuda")

    def run(x):
        x = x.detach().requires_grad_(True)
        if which == "tokens":
            lp = token_log_probs(x, y)
            return [lp.detach(), torch.autograd.grad(lp, x, torch.ones_like(lp))[0]]
        if which == "pairs":
            loss, a, b = preference_loss(x, y, ref, 0.01)
            return [loss.detach(), a, b, torch.autograd.grad(loss, x, scale)[0]]
        loss, lp = policy_loss(x, y, None, adv, grad_scale=1.0 if which == "at once" else None)
        return [loss.detach(), lp, torch.autograd.grad(loss, x, scale)[0]]

    buf = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(buf)
    for x in xs + xs[:1]:
        buf.copy_(x)
        graph.replay()
        got = [o.clone() for o in outs]
        want = run(x)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_refusals_on_the_gpu():
    x, y, _ = make((4, 5), 12, torch.float32)
    x = x.cuda()
    with pytest.raises(ValueError, match="labels are on"):
        token_log_probs(x, y)
    y = y.cuda()
    with pytest.raises(ValueError, match="ref_log_probs is on"):
        preference_loss(x, y, torch.zeros(4))
    with pytest.raises(ValueError, match="cu_seqlens are on"):
        sequence_log_probs(x.view(20, 12), y.view(20), torch.tensor([0, 20], dtype=torch.int32))
    with pytest.raises(ValueError, match="old_log_probs is on"):
        policy_loss(x, y, torch.zeros(4, 5), torch.zeros(4, device="cuda"))
    with pytest.raises(ValueError, match="grad_scale"):
        policy_loss(x, y, None, torch.zeros(4, device="cuda"), grad_scale=torch.ones(1))


def test_a_change_in_place_is_noticed():
    x, y, _ = make((4, 5), 12, torch.float32)
    w = torch.ones((), device="cuda", requires_grad=True)
    x = x.cuda() * w
    lp = token_log_probs(x, y.cuda())
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        lp.sum().backward()


def test_gradients_are_differentiable_once():
    x, y, _ = make((4, 5), 12, torch.float32, ignored=0)
    x = x.cuda().requires_grad_(True)
    w = torch.ones(4, 5, device="cuda", requires_grad=True)
    g = torch.autograd.grad(token_log_probs(x, y.cuda()), x, w, create_graph=True)[0]
    assert torch.isfinite(g).all()
    with pytest.raises(RuntimeError, match="once only"):
        g.sum().backward()


def test_outputs_without_a_gradient():
    """Rewards and log-probabilities are not differentiable; a loss that nothing asks for leaves no gradient."""
    x, y, _ = make((4, 5), 12, torch.float32, ignored=0)
    x = x.cuda().requires_grad_(True)
    loss, chosen, rejected = preference_loss(x, y.cuda(), torch.zeros(4, device="cuda"))
    assert loss.requires_grad and not chosen.requires_grad and not rejected.requires_grad
    loss, lp = policy_loss(x, y.cuda(), None, torch.ones(4, device="cuda"))
    assert loss.requires_grad and not lp.requires_grad
    (chosen.sum() + rejected.sum() + lp.sum() + x.sum()).backward()
    assert (x.grad == 1).all()
    with torch.no_grad():
        assert not policy_loss(x, y.cuda(), None, torch.ones(4, device="cuda"))[0].requires_grad


def test_gradients_add_up_over_calls():
    """Two calls on one leaf, a loss of both: AccumulateGrad and the sum of the two gradients."""
    x, y, _ = make((4, 5), 300, torch.float32, ignored=0)
    ref = torch.zeros(4, device="cuda")
    a, b = x.cuda().requires_grad_(True), x.cuda().requires_grad_(True)
    la, lb = preference_loss(a, y.cuda(), ref)[0], policy_loss(a, y.cuda(), None, ref + 1, grad_scale=1.0)[0]
    (la + lb).backward()
    want = torch.autograd.grad(preference_loss(b, y.cuda(), ref)[0], b)[0] + torch.autograd.grad(policy_loss(b, y.cuda(), None, ref + 1)[0], b)[0]
    # fp32 sums of two values under 1, each within some half steps
    torch.testing.assert_close(a.grad, want, rtol=0, atol=8 * 2 ** -24)


def test_rows_beyond_32_bits():
    """Rows that begin, and gradients that lie, more than 2^31 elements from the first."""
    g = torch.Generator().manual_seed(0)
    few = torch.randn(2, 300, generator=g)
    base = torch.empty(2_200_000_300, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((2, 300), (2_200_000_000, 1))
    x.copy_(few)
    y = torch.tensor([3, 299])
    few = few.to(torch.bfloat16)
    near(token_log_probs(x, y.cuda()), oracle.log_probs(few.double(), y), oracle.lp_bound(few, y))
    del base, x
    rows, vocab = 70000, 32000
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    last = (torch.randn(2, vocab, generator=g) * 2).to(torch.bfloat16)
    x[-2:] = last.cuda()
    y = torch.full((rows,), -100, device="cuda")
    y[-2:] = torch.tensor([5, 31999], device="cuda")
    x.requires_grad_(True)
    dx = grad_of(token_log_probs(x, y), x, torch.ones(rows))
    l64 = last.double().requires_grad_(True)
    lp = oracle.log_probs(l64, y[-2:].cpu())
    near(dx[-2:], torch.autograd.grad(lp.sum(), l64)[0], oracle.grad_bound(last, y[-2:].cpu(), torch.ones(2), torch.bfloat16))
    assert not dx[:-2].any()


def test_a_ratio_that_overflows_and_one_of_nothing():
    """The clip's and the kernel's own sides of an infinite ratio, and of a token of probability 0, as the CPU path has them."""
    x = torch.zeros(1, 3, 4)
    x[0, 0, 1] = -math.inf
    y = torch.tensor([[1, 2, 0]])
    for old in (None, torch.tensor([[0.0, -200.0, -1.3]])):
        for scale in (None, 1.0):
            out = []
            for device in ("cpu", "cuda"):
                z = x.to(device).requires_grad_(True)
                loss, lp = policy_loss(z, y.to(device), None if old is None else old.to(device), torch.ones(1, device=device), grad_scale=scale)
                out.append([loss.detach().cpu(), lp.cpu(), torch.autograd.grad(loss, z)[0].cpu()])
            for a, b in zip(*out):
                assert not torch.isnan(a).any()
                torch.testing.assert_close(a, b, rtol=0, atol=8 * 2 ** -24)


def test_no_sequences():
    """An empty batch has no log-probabilities and an empty gradient, as on the CPU."""
    for device in ("cpu", "cuda"):
        x = torch.zeros(0, 3, 7, device=device, requires_grad=True)
        y = torch.zeros(0, 3, dtype=torch.long, device=device)
        for average in (False, True):
            out = sequence_log_probs(x, y, average=average)
            assert out.shape == (0,) and out.dtype == torch.float32
            assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape
        assert token_log_probs(x, y).shape == (0, 3)
        with pytest.raises(ValueError, match="needs"):
            preference_loss(x, y, torch.zeros(0, device=device))
        with pytest.raises(ValueError, match="needs"):
            policy_loss(x, y, None, torch.zeros(0, device=device))


@pytest.mark.parametrize("t", [0.7, 1.0, 1.3])
def test_both_ways_of_the_policy_gradient_round_alike(t):
    """Logits far apart, where an exponent's base that is off shows. A row has one pack a lane both ways, so its sum and
    then each step of its gradient are the same: so are all bits."""
    x = (torch.randn(4, 16, 256, generator=torch.Generator().manual_seed(7)) * 30).cuda().requires_grad_(True)
    y = x.detach().argmax(-1)
    adv, out = torch.ones(4, device="cuda"), []
    for scale in (None, 1.0):
        loss, lp = policy_loss(x, y, None, adv, temperature=t, reduction="sum", grad_scale=scale)
        out.append([lp, torch.autograd.grad(loss, x, torch.ones((), device="cuda"))[0]])
    for a, b in zip(*out):
        assert torch.equal(a, b)


@pytest.mark.parametrize("scale", [None, 1.0])
def test_advantages_of_as_many_sequences_as_tokens(scale):
    """[sequences] is the labels' shape there and goes by token; [sequences, 1] goes by sequence: the CPU path's results."""
    x, y, g = make((5,), 6, torch.float32, ignored=0)
    adv, cu = torch.randn(5, generator=g), torch.tensor([0, 2, 2, 3, 4, 5], dtype=torch.int32)
    old = oracle.log_probs(x.double(), y).float() + 0.1 * torch.randn(5, generator=g)
    for a in (adv, adv[:, None]):
        out = []
        for device in ("cpu", "cuda"):
            z = x.to(device).requires_grad_(True)
            loss, _ = policy_loss(z, y.to(device), old.to(device), a.to(device), cu_seqlens=cu.to(device), grad_scale=scale)
            out.append([loss.detach().cpu(), torch.autograd.grad(loss, z)[0].cpu()])
        for a, b in zip(*out):
            # losses and slopes of up to 3, in fp32 on both sides
            torch.testing.assert_close(a, b, rtol=0, atol=64 * 2 ** -24)
