"""FusedAdam8bit on the CPU path: its codes, the mean of its rounding, the step against 64 bits, checkpoints, refusals."""

import copy
import math

import pytest
import torch

from apex_amd.optimizers import FusedAdam8bit
from apex_amd.optimizers.fused_adam_8bit import _decode, _encode, _mix, _random_bits

TABLE = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 ... 448


def test_random_bits_are_even():
    """Both halves of 2^17 consecutive elements' bits, and two steps' against each other. Counts of 256 bins of 512
    expected: a deviation over 6 sigma (136) has odds under 1e-6 for all of them together."""
    a, b = _random_bits(3, 10, 5, 1 << 17), _random_bits(3, 11, 5, 1 << 17)
    for bits in (a & 0xFFFF, a >> 16, (a ^ b) & 0xFFFF, (a ^ b) >> 16, (a & 0xFFFF) ^ (a >> 16), (a[1:] ^ a[:-1]) >> 16):
        counts = torch.bincount(bits >> 8, minlength=256)
        assert (counts - 512).abs().max() < 136
    assert _mix(0) == 0 and 0 < _mix(1) <= 0xFFFFFFFF


@pytest.mark.parametrize("root", [False, True])
def test_codes_are_neighbours(root):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(1000, generator=g) * torch.exp(4 * torch.randn(1000, generator=g))
    x = x.abs() if root else x
    x[5:9] = 0
    codes, scales = _encode(x, torch.rand(1000, generator=g), root)
    assert codes.shape == x.shape and scales.shape == (8,)
    for b in range(8):
        part = x[128 * b: 128 * b + 128].double()
        assert scales[b] == (part.abs().max().float() / 448)
        y = (part / scales[b].double()).abs().clamp(max=448)
        got = codes[128 * b: 128 * b + 128].double()
        assert ((got == 0) | (torch.sign(got) == torch.sign(part))).all()
        # a y within a rounding of a code may count as on either side of it
        lo = TABLE[(torch.searchsorted(TABLE, y * (1 - 2.0 ** -20), right=True) - 1).clamp(min=0)]
        hi = TABLE[torch.searchsorted(TABLE, y * (1 + 2.0 ** -20)).clamp(max=126)]
        assert ((got.abs() >= lo) & (got.abs() <= hi)).all()
        if root:
            assert ((got > 0) == (part > 0)).all()


@pytest.mark.parametrize("root", [False, True])
def test_rounding_keeps_the_mean(root):
    """Over u = (k + 0.5) / 65536 for every k the mean is exact to a part of 65536 of the codes' distance."""
    u = (torch.arange(65536) + 0.5) / 65536
    for value in (447.9, 300.0, 17.3, 1.01, 0.02, 0.0021):
        x = torch.full((65536,), value)
        x[::128] = 448.0  # each block's scale is 1
        codes, _ = _encode(x, u, root)
        got = codes.double()[torch.arange(65536) % 128 != 0]
        power = 2 if root else 1
        i = torch.searchsorted(TABLE, value)
        gap = TABLE[i] ** power - TABLE[i - 1] ** power
        # the 512 left out are evenly spread over u: they move the mean by at most one part in 128 of u's own spacing
        mean = (got ** power).mean() if root else got.mean()
        assert abs(mean - float(torch.tensor(value)) ** power) < gap * 2e-3
    tiny = torch.full((128,), 1e-5)
    tiny[0] = 448.0
    codes, _ = _encode(tiny, torch.full((128,), 0.999), root)
    assert (codes.float()[1:] == (2.0 ** -9 if root else 0.0)).all()


def test_a_slow_average_moves():
    """With beta2 = 0.995 the second moment follows a gradient that becomes ten times smaller: its root falls by 0.25% a
    step where codes are 6% and more apart, so to nearest it would stay."""
    p = torch.nn.Parameter(torch.zeros(4096))
    opt = FusedAdam8bit([p], lr=0.0, betas=(0.9, 0.995))
    v, sizes = 0.0, [1.0] * 100 + [0.1] * 400
    for s in sizes:
        p.grad = torch.full((4096,), s)
        v = 0.995 * v + 0.005 * s * s
        opt.step()
    st = opt.state[p]
    got = (_decode(st["exp_avg_sq"], st["exp_avg_sq_scale"]).double() ** 2).mean()
    # elements wander by some tenths of v, each for itself: the mean of 4096 by under 1%
    assert abs(got / v - 1) < 0.05


def reference_step(p, g, m, r, step, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, wd=0.0, l2=False, bias=True):
    p, g = p.double(), g.double()
    if l2:
        g = g + wd * p
    m = betas[0] * m.double() + (1 - betas[0]) * g
    v = betas[1] * r.double() ** 2 + (1 - betas[1]) * g * g
    a = m / (1 - betas[0] ** step if bias else 1)
    b = (v / (1 - betas[1] ** step if bias else 1)).sqrt() + eps
    return p - lr * (a / b + (0.0 if l2 else wd * p)), m, v.sqrt()


@pytest.mark.parametrize("l2,bias,master", [(False, True, False), (True, False, False), (False, True, True)])
def test_steps_against_64_bits(l2, bias, master):
    g = torch.Generator().manual_seed(1)
    dtype = torch.bfloat16 if master else torch.float32
    shapes = [(3, 50), (1,), (128,), (0,), (129,)]
    params = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype)) for s in shapes]
    opt = FusedAdam8bit(params, lr=1e-2, weight_decay=0.1, adam_w_mode=not l2, bias_correction=bias, master_weights=master)
    for step in range(1, 4):
        old = []
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(dtype)
            st = opt.state[p]
            old.append([p.detach().clone(), torch.zeros(p.shape), torch.zeros(p.shape)] if not st else
                       [st.get("master_param", p.detach()).clone()] + [_decode(st[k].view(-1), st[k + "_scale"]).view(p.shape) for k in ("exp_avg", "exp_avg_sq")])
        opt.step()
        for p, (w, m, r) in zip(params, old):
            want, m, r = reference_step(w, p.grad, m, r, step, wd=0.1, l2=l2, bias=bias)
            st = opt.state[p]
            # fp32: under 20 half steps of a weight of 4 and a step of lr * (4 + 0.4)
            torch.testing.assert_close(st.get("master_param", p.detach()).double(), want, rtol=0, atol=20 * 2 ** -24 * 8)
            if master:
                assert torch.equal(p.detach(), st["master_param"].to(dtype))
            for x, k in ((m, "exp_avg"), (r, "exp_avg_sq")):
                got = _decode(st[k].view(-1), st[k + "_scale"]).view(p.shape).double()
                # the code above or below: within one distance, 1/8 of the value, or the smallest, 2^-9 of the scale
                far = x.abs() / 8 + (st[k + "_scale"].max().double() * 2 ** -9 if p.numel() else 0)
                assert ((got - x).abs() <= far * 1.0001).all()


def test_not_finite_stays_where_it_is():
    p = torch.nn.Parameter(torch.ones(300))
    opt = FusedAdam8bit([p], lr=1e-2)
    p.grad = torch.full((300,), 0.5)
    p.grad[7], p.grad[200] = math.inf, math.nan
    opt.step()
    bad = torch.zeros(300, dtype=torch.bool)
    bad[7] = bad[200] = True
    for k in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(torch.isnan(opt.state[p][k].float()), bad)
        assert torch.isfinite(opt.state[p][k + "_scale"]).all()
    assert torch.equal(torch.isfinite(p.detach()), ~bad)


def test_layouts_and_groups():
    """A transposed weight's elements are met in memory order; a gradient of another layout is the same gradient."""
    g = torch.Generator().manual_seed(2)
    w, d = torch.randn(20, 30, generator=g), torch.randn(20, 30, generator=g)
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.t().contiguous().t())
    assert b.stride() == (1, 20)
    for p in (a, b):
        opt = FusedAdam8bit([{"params": [p], "lr": 0.1}, {"params": []}], weight_decay=0.1)
        p.grad = d.clone() if p is a else d.t().contiguous().t()
        opt.step()
    torch.testing.assert_close(a.detach(), b.detach(), rtol=1e-6, atol=1e-6)
    c = torch.nn.Parameter(w.t().contiguous().t())
    opt2 = FusedAdam8bit([c], lr=0.1, weight_decay=0.1)
    c.grad = d.clone()
    opt2.step()
    assert torch.equal(b.detach(), c.detach())


@pytest.mark.parametrize("master", [False, True])
def test_a_checkpoint_goes_on_bit_for_bit(master):
    g = torch.Generator().manual_seed(3)
    start = torch.randn(5, 77, generator=g).to(torch.bfloat16 if master else torch.float32)
    grads = [torch.randn(5, 77, generator=g).to(start.dtype) for _ in range(4)]

    def go(opt, p, gs):
        for x in gs:
            p.grad = x.clone()
            opt.step()

    p = torch.nn.Parameter(start.clone())
    opt = FusedAdam8bit([p], lr=1e-2, master_weights=master, seed=9)
    go(opt, p, grads[:2])
    saved, q = copy.deepcopy(opt.state_dict()), torch.nn.Parameter(p.detach().clone())
    go(opt, p, grads[2:])
    other = FusedAdam8bit([q], lr=5.0, master_weights=master, seed=9)
    other.load_state_dict(saved)
    st = other.state[q]
    assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["exp_avg_scale"].dtype == torch.float32
    assert not master or st["master_param"].dtype == torch.float32
    go(other, q, grads[2:])
    assert torch.equal(p.detach(), q.detach())
    for k in st:
        assert torch.equal(opt.state[p][k].view(torch.uint8), other.state[q][k].view(torch.uint8))


def test_refusals():
    from apex_amd.optimizers import FusedAdam

    w = torch.nn.Parameter(torch.zeros(3))
    w.grad = torch.ones(3)
    other = FusedAdam([w])
    other.step()
    with pytest.raises(ValueError, match="exp_avg_scale"):
        FusedAdam8bit([w]).load_state_dict(other.state_dict())
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(RuntimeError, match="AMSGrad"):
        FusedAdam8bit([p], amsgrad=True)
    with pytest.raises(ValueError, match="betas"):
        FusedAdam8bit([p], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="eps"):
        FusedAdam8bit([p], eps=-1.0)
    d = torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))
    d.grad = torch.zeros_like(d)
    with pytest.raises(RuntimeError, match="fp16/bf16/fp32"):
        FusedAdam8bit([d]).step()
    e = torch.nn.Embedding(5, 3, sparse=True)
    e(torch.tensor([1])).sum().backward()
    with pytest.raises(RuntimeError, match="sparse"):
        FusedAdam8bit(e.parameters()).step()
    s = torch.nn.Parameter(torch.zeros(4, 6)[:, :3])
    s.grad = torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match="dense"):
        FusedAdam8bit([s]).step()


@pytest.mark.parametrize("unscale", [False, True])
def test_a_scaler_that_has_unscaled_already(unscale):
    """unscale_, clip, step: the step is that of the true gradients, bit for bit (the scale is a power of two), at an eps
    that tells their size; one that is not finite skips it and does not count."""
    g = torch.Generator().manual_seed(4)
    start = [torch.randn(s, generator=g) for s in ((3, 50), (129,))]
    args = dict(lr=1e-2, eps=1e-2, capturable=True, master_weights=True)
    pa, pb = ([torch.nn.Parameter(w.clone()) for w in start] for _ in range(2))
    a, b = (FusedAdam8bit([{"params": p[:1]}, {"params": p[1:]}], **args) for p in (pa, pb))
    scaler = torch.amp.GradScaler("cpu", init_scale=1024.0, growth_interval=1000)
    scaler.scale(torch.zeros(()))
    for step in range(3):
        for p, q in zip(pa, pb):
            d = 0.02 * torch.randn(p.shape, generator=g)
            p.grad, q.grad = d * 1024, d
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
        else:
            b.step()
        assert [int(x["step"]) for x in a.param_groups] == [(1, 1, 2)[step]] * 2
        for p, q in zip(pa, pb):
            assert torch.equal(p, q)
            for k in a.state[p]:
                assert torch.equal(a.state[p][k].view(torch.uint8), b.state[q][k].view(torch.uint8))


def test_a_scaler_is_asked_once_for_a_step():
    """Whatever the number of groups: each question reads and writes all gradients. After unscale_ it is not asked."""
    params = [torch.nn.Parameter(torch.ones(5)) for _ in range(3)]
    opt = FusedAdam8bit([{"params": [p]} for p in params], capturable=True)
    scaler, asked = torch.amp.GradScaler("cpu", init_scale=4.0), []
    scaler.scale(torch.zeros(()))
    check = scaler._check_inf_per_device
    scaler._check_inf_per_device = lambda o: (asked.append(o), check(o))[1]
    for unscale, times in ((False, 1), (True, 1)):
        for p in params:
            p.grad = torch.ones(5)
        if unscale:
            scaler.unscale_(opt)
        scaler.step(opt)
        scaler.update()
        assert len(asked) == times
    assert [int(g["step"]) for g in opt.param_groups] == [2, 2, 2]


def test_what_one_device_found_holds_for_all():
    """Params on several devices: one gradient that is not finite skips the step of each (the scaler's record of another
    device is made up here)."""
    from torch.amp.grad_scaler import OptState

    p = torch.nn.Parameter(torch.ones(5))
    opt = FusedAdam8bit([p], capturable=True)
    scaler = torch.amp.GradScaler("cpu")
    scaler.scale(torch.zeros(()))
    for found in (1.0, 0.0):
        p.grad = torch.ones(5)
        scaler._per_optimizer_states[id(opt)] = {
            "stage": OptState.UNSCALED,
            "found_inf_per_device": {torch.device("cpu"): torch.tensor(0.0), torch.device("cpu", 1): torch.tensor(found)},
        }
        opt.step(grad_scaler=scaler)
        assert torch.equal(p.detach(), torch.ones(5)) == bool(found) and int(opt.param_groups[0]["step"]) == 1 - int(found)


def test_each_group_has_a_learning_rate_of_its_own():
    """A schedule writes tensor rates in place: one that two groups share would hold the last group's value."""
    params = [torch.nn.Parameter(torch.zeros(5)) for _ in range(4)]
    opt = FusedAdam8bit([{"params": params[:1]}, {"params": params[1:2]}, {"params": params[2:3], "lr": 0.5}], lr=1e-2, capturable=True)
    opt.add_param_group({"params": params[3:]})
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, [lambda e, f=f: f for f in (1.0, 0.1, 0.01, 0.001)])
    want = [1e-2, 1e-3, 5e-3, 1e-5]

    def rates(o):
        assert all(torch.is_tensor(g["lr"]) and g["lr"].dtype == torch.float32 for g in o.param_groups)
        return [g["lr"].item() for g in o.param_groups]

    assert rates(opt) == pytest.approx(want)
    for p in params:
        p.grad = torch.ones(5)
    opt.step()
    # m / root(v) is 1 in the first step
    assert [-p[0].item() for p in params] == pytest.approx(want, rel=1e-5)
    schedule.step()
    assert rates(opt) == pytest.approx(want)
    other = FusedAdam8bit([{"params": [torch.nn.Parameter(torch.zeros(5))]} for _ in range(4)], lr=1.0, capturable=True)
    other.load_state_dict(opt.state_dict())
    assert rates(other) == pytest.approx(want)
    other.param_groups[0]["lr"].fill_(7.0)
    assert rates(other) == pytest.approx([7.0] + want[1:])
    # a checkpoint of groups that share one tensor
    saved = opt.state_dict()
    for g in saved["param_groups"]:
        g["lr"] = opt.param_groups[0]["lr"]
    other.load_state_dict(saved)
    other.param_groups[0]["lr"].fill_(7.0)
    assert rates(other) == pytest.approx([7.0, 1e-2, 1e-2, 1e-2])


def test_a_learning_rate_that_the_caller_holds():
    """A tensor that the caller gives is used as it is, by every group without a rate of its own: what torch does."""
    params = [torch.nn.Parameter(torch.zeros(5)) for _ in range(2)]
    lr = torch.tensor(1e-2)
    opt = FusedAdam8bit([{"params": [p]} for p in params], lr=lr, capturable=True)
    lr.fill_(3e-3)
    for p in params:
        p.grad = torch.ones(5)
    opt.step()
    assert [-p[0].item() for p in params] == pytest.approx([3e-3, 3e-3], rel=1e-5)


def test_a_checkpoint_without_masters_gets_them_and_one_with_them_loses_them():
    """master_weights is the loading optimizer's to say. 2 - 1e-5 is no bf16: without masters the weight never moves."""
    def go(opt, p, steps):
        for _ in range(steps):
            p.grad = torch.ones_like(p)
            opt.step()

    def new(master):
        p = torch.nn.Parameter(torch.ones(200, dtype=torch.bfloat16))
        return p, FusedAdam8bit([p], lr=1e-5, master_weights=master)

    p, without = new(False)
    go(without, p, 2)
    q, opt = new(True)
    opt.load_state_dict(without.state_dict())
    with torch.no_grad():
        q.fill_(2.0)  # the weights may be loaded after the optimizer
    go(opt, q, 5)
    # the same from a checkpoint that has them
    saved = without.state_dict()
    saved["state"][0] = saved["state"][0] | {"master_param": torch.full((200,), 2.0)}
    w, other = new(True)
    other.load_state_dict(saved)
    go(other, w, 5)
    master = opt.state[q]["master_param"]
    assert master.dtype == torch.float32 and (master < 2.0 - 3e-5).all()
    assert torch.equal(master, other.state[w]["master_param"]) and torch.equal(q.detach(), master.bfloat16())
    r, back = new(False)
    back.load_state_dict(opt.state_dict())
    go(back, r, 2)
    assert "master_param" not in back.state[r] and torch.equal(r.detach(), torch.ones(200, dtype=torch.bfloat16))
    assert "master_param" in opt.state[q]


@pytest.mark.parametrize("capturable", [False, True])
def test_a_checkpoint_brings_its_seed(capturable):
    """The random numbers go on as they would have, whatever seed the loading optimizer was made with; a checkpoint
    from before seeds were kept leaves it its own."""
    g = torch.Generator().manual_seed(5)
    grads = [torch.randn(300, generator=g) for _ in range(4)]

    def go(opt, p, gs):
        for x in gs:
            p.grad = x.clone()
            opt.step()

    def new(seed):
        p = torch.nn.Parameter(torch.zeros(300))
        return p, FusedAdam8bit([p], lr=1e-2, seed=seed, capturable=capturable)

    p, opt = new(9)
    go(opt, p, grads[:2])
    saved, start = copy.deepcopy(opt.state_dict()), p.detach().clone()
    go(opt, p, grads[2:])
    old = copy.deepcopy(saved)
    assert old["param_groups"][0].pop("seed") == 9
    for state, seed in ((saved, 0), (old, 9)):
        q, other = new(seed)
        with torch.no_grad():
            q.copy_(start)
        other.load_state_dict(state)
        go(other, q, grads[2:])
        assert torch.equal(p.detach(), q.detach())
        for k in opt.state[p]:
            assert torch.equal(opt.state[p][k].view(torch.uint8), other.state[q][k].view(torch.uint8))


def test_a_checkpoint_of_other_params_is_refused():
    """Codes are met in memory order with a scale for each 128: those of another shape or layout, or without all their
    scales, would be taken for other elements'. Dimensions of one element have no layout."""
    w = torch.randn(8, 3, 5, 5, generator=torch.Generator().manual_seed(6))

    def saved(p):
        opt = FusedAdam8bit([p])
        p.grad = torch.ones_like(p)
        opt.step()
        return opt.state_dict()

    last = torch.nn.Parameter(w.to(memory_format=torch.channels_last))
    for p, q in ((last, w), (torch.nn.Parameter(w.clone()), w.to(memory_format=torch.channels_last)),
                 (torch.nn.Parameter(w.reshape(3, 8, 5, 5)), w)):
        opt = FusedAdam8bit([torch.nn.Parameter(q.clone())])
        with pytest.raises(ValueError, match="layout"):
            opt.load_state_dict(saved(p))
        assert not opt.state
    for name, change in (("exp_avg_scale", lambda x: x[:-1]), ("exp_avg_sq_scale", lambda x: x.double()),
                         ("exp_avg", lambda x: x.float()), ("exp_avg_sq", lambda x: x.view(torch.uint8))):
        state = saved(torch.nn.Parameter(w.clone()))
        state["state"][0][name] = change(state["state"][0][name])
        with pytest.raises(ValueError, match=name):
            FusedAdam8bit([torch.nn.Parameter(w.clone())]).load_state_dict(state)
    column = torch.randn(200, 1)
    other = torch.nn.Parameter(column.as_strided((200, 1), (1, 7)))
    state = saved(torch.nn.Parameter(column.clone()))
    opt = FusedAdam8bit([other])
    opt.load_state_dict(state)
    other.grad = torch.ones(200, 1)
    opt.step()
    assert opt.state[other]["exp_avg"].shape == (200, 1)
