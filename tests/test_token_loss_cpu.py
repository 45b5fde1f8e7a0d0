"""Token losses on the CPU path: values and gradients against 64 bits and against differences, and refusals."""

import math

import pytest
import torch

import token_loss_oracle as oracle
from apex_amd.contrib.xentropy import policy_loss, preference_loss, sequence_log_probs, token_log_probs

CU = [1, 4, 4, 9, 13]  # a token before the first sequence, an empty one, and one behind the last of 14


def make(lead, vocab, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*lead, vocab, generator=g) * 2).to(dtype)
    y = torch.randint(0, vocab, lead, generator=g)
    y[torch.rand(lead, generator=g) < 0.3] = -100
    return x, y, g


def grads(loss64, x64, loss, x):
    """Gradients in 64 bits and here."""
    return torch.autograd.grad(loss64, x64)[0], torch.autograd.grad(loss, x)[0].double()


def both(x):
    return x.double().requires_grad_(True), x.clone().requires_grad_(True)


# fp32 torch: 20 half steps of values of about 20 (logits, log sums), and of sums of 14 of them
TOL = dict(rtol=0, atol=20 * 2 ** -24 * 20 * 14)


@pytest.mark.parametrize("lead,vocab,t", [((3, 5), 11, 1.0), ((7,), 1, 0.5), ((2, 3, 4), 33, 2.0)])
def test_token_log_probs(lead, vocab, t):
    x, y, g = make(lead, vocab)
    x64, x = both(x)
    want, got = oracle.log_probs(x64, y, temperature=t), token_log_probs(x, y, temperature=t)
    torch.testing.assert_close(got.double(), want, **TOL)
    w = torch.randn(lead, generator=g)
    a, b = grads((want * w).sum(), x64, (got * w).sum(), x)
    torch.testing.assert_close(b, a, **TOL)


def test_ignored_rows_may_hold_anything():
    x, y, _ = make((2, 6), 9)
    y[:, 0], y[:, 1] = -100, 3
    x[0, 0], x[1, 0] = math.nan, math.inf
    x.requires_grad_(True)
    lp = token_log_probs(x, y)
    lp.sum().backward()
    assert (lp[y == -100] == 0).all() and torch.isfinite(lp).all()
    assert (x.grad[y == -100] == 0).all() and torch.isfinite(x.grad).all()


@pytest.mark.parametrize("average", [False, True])
@pytest.mark.parametrize("cu", [None, CU])
def test_sequence_log_probs(cu, average):
    x, y, g = make((4, 5) if cu is None else (14,), 12)
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    x64, x = both(x)
    want = oracle.sums(oracle.log_probs(x64, y), y, cu=cu, average=average)
    got = sequence_log_probs(x, y, c, average=average)
    torch.testing.assert_close(got.double(), want, **TOL)
    w = torch.randn(4, generator=g)
    a, b = grads((want * w).sum(), x64, (got * w).sum(), x)
    torch.testing.assert_close(b, a, **TOL)
    if cu is not None:
        assert (b[0] == 0).all() and (b[13] == 0).all()


@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("ipo", 0.0), ("hinge", 0.0)])
@pytest.mark.parametrize("cu,average", [(None, False), (CU, True)])
def test_preference_loss(kind, smoothing, cu, average):
    x, y, g = make((4, 5) if cu is None else (14,), 12)
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    ref = torch.randn(4, generator=g) - 5
    x64, x = both(x)
    want, gain = oracle.preference(x64, y, ref, 0.3, smoothing, kind, average, cu)
    loss, chosen, rejected = preference_loss(x, y, ref, 0.3, smoothing, kind, average, c)
    scale = 2 * (20 / 0.3 + 40) if kind == "ipo" else 1  # the square's slope
    torch.testing.assert_close(loss.double(), want, rtol=0, atol=TOL["atol"] * scale)
    torch.testing.assert_close(torch.cat([chosen, rejected]).double(), gain, **TOL)
    assert not chosen.requires_grad and not rejected.requires_grad
    a, b = grads(want, x64, loss, x)
    torch.testing.assert_close(b, a, rtol=0, atol=TOL["atol"] * scale)


@pytest.mark.parametrize("reduction", ["token", "sequence", "sum", "none"])
@pytest.mark.parametrize("cu,by_row,kl,on_policy", [(None, False, 0.1, False), (None, True, 0.0, True), (CU, False, 0.0, False), (CU, True, 0.2, False)])
def test_policy_loss(reduction, cu, by_row, kl, on_policy):
    x, y, g = make((4, 5) if cu is None else (14,), 12)
    c = None if cu is None else torch.tensor(cu, dtype=torch.int32)
    lp = oracle.log_probs(x.double(), y).float()
    old = None if on_policy else lp + 0.3 * torch.randn(y.shape, generator=g)
    ref = lp + torch.randn(y.shape, generator=g) if kl else None
    adv = torch.randn(y.shape if by_row else (4,), generator=g)
    x64, x = both(x)
    args = dict(kl=kl, reduction=reduction, cu=cu, high=0.3, temperature=1.0)
    want, lp64 = oracle.policy(x64, y, old, adv, ref, **args)
    loss, got = policy_loss(x, y, old, adv, ref, clip_eps_high=0.3, kl_coef=kl, reduction=reduction, cu_seqlens=c)
    torch.testing.assert_close(loss.double(), want, **TOL)
    torch.testing.assert_close(got.double(), lp64, **TOL)
    w = torch.randn(want.shape, generator=g)
    a, b = grads((want * w).sum(), x64, (loss * w).sum(), x)
    torch.testing.assert_close(b, a, **TOL)


@pytest.mark.parametrize("kind", ["sigmoid", "hinge"])
def test_a_rejected_answer_that_cannot_be(kind):
    """A rejected token of probability 0: the pair is as right as can be, and asks for nothing."""
    x = torch.zeros(2, 3, 5)
    x[1, 1, 4] = -math.inf
    y = torch.tensor([[0, 1, 2], [3, 4, 0]])
    x.requires_grad_(True)
    loss, _, rejected = preference_loss(x, y, torch.zeros(2), loss_type=kind)
    assert loss == 0 and rejected[0] == -math.inf
    loss.backward()
    assert (x.grad == 0).all()


def test_gradients_against_differences():
    """The formulas' gradients, in 64 bits, against central differences: what the other tests hold the kernels to."""
    x, y, g = make((4, 3), 6)
    x = x.double().requires_grad_(True)
    lp = oracle.log_probs(x.detach(), y)
    old, ref = lp + 0.05 * torch.randn(y.shape, generator=g), lp + 0.3
    adv = torch.randn(4, generator=g)
    assert torch.autograd.gradcheck(lambda x: oracle.policy(x, y, old, adv, ref, kl=0.1)[0], (x,))
    assert torch.autograd.gradcheck(lambda x: oracle.preference(x, y, torch.zeros(4), smoothing=0.1)[0], (x,))


def test_refusals():
    x, y, _ = make((4, 5), 12)
    ok = torch.zeros(4, 5)
    with pytest.raises(TypeError, match="logits"):
        token_log_probs(x.double(), y)
    with pytest.raises(TypeError, match="labels"):
        token_log_probs(x, y.float())
    with pytest.raises(ValueError, match="labels must have shape"):
        token_log_probs(x, y[:, :4])
    with pytest.raises(ValueError, match="vocabulary"):
        token_log_probs(x[..., :0], y)
    for t in (0.0, -1.0, 1e-7, 1e7, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            token_log_probs(x, y, temperature=t)
    with pytest.raises(ValueError, match="cu_seqlens"):
        sequence_log_probs(x.view(20, 12), y.view(20))
    with pytest.raises(ValueError, match="1-D"):
        sequence_log_probs(x, y, torch.tensor([0, 5], dtype=torch.int32))
    with pytest.raises(ValueError, match="int32"):
        sequence_log_probs(x.view(20, 12), y.view(20), torch.tensor([0, 5]))
    with pytest.raises(ValueError, match="pairs"):
        preference_loss(x[:3], y[:3], torch.zeros(3))
    with pytest.raises(ValueError, match="pairs"):
        preference_loss(x[:, :0], y[:, :0], torch.zeros(4))
    with pytest.raises(ValueError, match="ref_log_probs must have shape"):
        preference_loss(x, y, torch.zeros(2))
    with pytest.raises(ValueError, match="loss_type"):
        preference_loss(x, y, torch.zeros(4), loss_type="other")
    with pytest.raises(ValueError, match="beta"):
        preference_loss(x, y, torch.zeros(4), beta=0.0)
    with pytest.raises(ValueError, match="label_smoothing"):
        preference_loss(x, y, torch.zeros(4), label_smoothing=0.5)
    with pytest.raises(ValueError, match="label_smoothing"):
        preference_loss(x, y, torch.zeros(4), label_smoothing=0.1, loss_type="ipo")
    with pytest.raises(ValueError, match="old_log_probs"):
        policy_loss(x, y, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="advantages"):
        policy_loss(x, y, ok, torch.zeros(5))
    with pytest.raises(TypeError, match="advantages"):
        policy_loss(x, y, ok, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="kl_coef needs"):
        policy_loss(x, y, ok, torch.zeros(4), kl_coef=0.1)
    with pytest.raises(ValueError, match="kl_coef"):
        policy_loss(x, y, ok, torch.zeros(4), ok, kl_coef=-0.1)
    with pytest.raises(ValueError, match="clip_eps"):
        policy_loss(x, y, ok, torch.zeros(4), clip_eps=1.5)
    with pytest.raises(ValueError, match="reduction"):
        policy_loss(x, y, ok, torch.zeros(4), reduction="mean")
    with pytest.raises(ValueError, match="grad_scale"):
        policy_loss(x, y, ok, torch.zeros(4), grad_scale=0.0)
    with pytest.raises(ValueError, match="grad_scale"):
        policy_loss(x, y, ok, torch.zeros(4), grad_scale=1.0, reduction="none")
    with pytest.raises(ValueError, match="token"):
        policy_loss(x[:, :0], y[:, :0], ok[:, :0], torch.zeros(4))


def test_a_ratio_that_overflows_and_one_of_nothing():
    """Where a clip holds a ratio of inf the gradient is 0, as where it holds any other; without old_log_probs the ratio is
    1, and its gradient that of lp, for a token of probability 0 too."""
    x = torch.zeros(1, 3, 4)
    x[0, 0, 1] = -math.inf
    x.requires_grad_(True)
    y = torch.tensor([[1, 2, 0]])
    p = torch.softmax(x.detach(), -1)
    want = (torch.nn.functional.one_hot(y, 4) - p) / 3  # of the mean of lp
    for a, reduction in ((1.0, "token"), (-2.0, "sequence"), (0.5, "sum")):
        adv = torch.full((1,), a)
        loss, lp = policy_loss(x, y, None, adv, reduction=reduction)
        n = 3 if reduction != "sum" else 1
        assert lp[0, 0] == -math.inf and loss == -a * 3 / n
        torch.testing.assert_close(torch.autograd.grad(loss, x)[0], -a * want * 3 / n, rtol=0, atol=8 * 2 ** -24)
    # exp(lp - old) is inf, in the middle token held at 1.2
    old = torch.tensor([[0.0, -200.0, -1.3]])
    loss, _ = policy_loss(x, y, old, torch.ones(1), reduction="none")
    assert loss[0, 0] == 0 and abs(loss[0, 1].item() + 1.2) < 4 * 2 ** -24
    dx = torch.autograd.grad(loss, x, torch.ones(1, 3))[0]
    assert (dx[0, :2] == 0).all() and torch.isfinite(dx).all() and dx[0, 2].abs().sum() > 0


def test_advantages_of_as_many_sequences_as_tokens():
    """[sequences] is the labels' shape there and goes by token; [sequences, 1] goes by sequence whatever their number."""
    cu = [0, 2, 2, 3, 4, 5]
    x, y, g = make((5,), 6)
    y = y.clamp(min=0)
    adv = torch.randn(5, generator=g)
    packed = torch.tensor(cu, dtype=torch.int32)
    old = oracle.log_probs(x.double(), y).float() + 0.1 * torch.randn(5, generator=g)
    rows = adv[torch.tensor([0, 0, 2, 3, 4])]  # what the sequences' are for the tokens
    for a, each in ((adv, adv), (adv[:, None], rows)):
        x64, mine = both(x)
        want, _ = oracle.policy(x64, y, old, each, cu=cu)
        got, _ = policy_loss(mine, y, old, a, cu_seqlens=packed)
        torch.testing.assert_close(got.double(), want, **TOL)
        wanted, dx = grads(want, x64, got, mine)
        torch.testing.assert_close(dx, wanted, **TOL)
    # a padded batch takes it too
    x, y, g = make((3, 4), 6)
    a = policy_loss(x, y, None, adv[:3])[0]
    assert torch.equal(a, policy_loss(x, y, None, adv[:3, None])[0])
    for bad in (adv[:4, None], adv[None, :3]):
        with pytest.raises(ValueError, match="advantages"):
            policy_loss(x, y, None, bad)
