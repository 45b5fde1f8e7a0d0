"""FusedAdam8bit on the GPU: its CPU path's state and weights over several steps, sizes, layouts, graphs, and a run."""

import math

import pytest
import torch

from apex_amd.optimizers import FusedAdam8bit
from apex_amd.optimizers.fused_adam_8bit import BLOCK, _decode

pytestmark = pytest.mark.gpu

# 1 to 129: around a block; 8191 to 8193, 20000: around a workgroup's part; 0: nothing
SIZES = [(1,), (7,), (8, 1), (127,), (128,), (129,), (0, 5), (8191,), (8192,), (8193,), (100, 200), (3, 5, 7)]


def make(sizes, dtype, seed=0, device="cpu", spread=3.0):
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(s, generator=g).to(dtype).to(device)) for s in sizes]

    def grads(step):
        g = torch.Generator().manual_seed(1000 * seed + step)
        for p in params:
            size = torch.exp(spread * torch.randn(p.shape, generator=g))
            p.grad = (torch.randn(p.shape, generator=g) * size * 1e-2).to(dtype).to(device)
    return params, grads


def codes(state, key):
    return state[key].detach().cpu().view(torch.uint8).to(torch.int32).view(-1)


def start_alike(a, b, pa, pb):
    """The CPU's optimizer goes on from what the GPU's holds."""
    for p, q in zip(pa, pb):
        q.detach().copy_(p.detach())
        for k, v in a.state[p].items():
            b.state[q][k] = v.detach().cpu().clone(memory_format=torch.preserve_format)


def l2_slack(b, pb, lr, wd):
    """With wd p added to g a small sum of large parts is off by 4 half steps of the parts, d. The step lr m / r has the
    slopes 0.1 / r and (m / r) (0.001 g / r^2) in g; m / r is under 40, and 0.001 g under 0.0316 r, so it is off by at
    most lr 1.4 d / r."""
    out = []
    for p in pb:
        st = b.state[p]
        w = st.get("master_param", p.detach()).double().view(-1)
        old = (_decode(st["exp_avg_sq"].view(-1), st["exp_avg_sq_scale"]) if st else torch.zeros(p.numel())).double()
        g = p.grad.double().view(-1)
        r = (0.999 * old ** 2 + 0.001 * (g + wd * w) ** 2).sqrt()
        out.append((lr * 1.4 * 4 * 2 ** -24 * ((wd * w).abs() + g.abs()) / r.clamp(min=1e-30)).view(p.shape))
    return out


def same(a, b, pa, pb, lr, dtype, slack=None):
    """One step from the same state. The kernel's arithmetic differs from torch's by a few half steps of fp32: a scale by
    at most 8 of them, and a code by one where a value lies within 8 of its threshold. Thresholds are 2^-3 of a value
    apart at least, so 2^-17 of all codes are expected to differ; 1 in 10^4 is allowed. A weight is rounded to its type
    (one whole step where that falls to another side) and its step, of at most lr * 40, is off by 16 half steps: m over
    the root of v is under 0.1 / sqrt(0.001) < 4 in one step, and a bias correction at most 10."""
    off, total = 0, 0
    for i, (p, q) in enumerate(zip(pa, pb)):
        s, t = a.state[p], b.state[q]
        assert s.keys() == t.keys()
        for k in ("exp_avg", "exp_avg_sq"):
            torch.testing.assert_close(s[k + "_scale"].cpu(), t[k + "_scale"].cpu(), rtol=8 * 2 ** -24, atol=1e-37)
            d = (codes(s, k) - codes(t, k)).abs()
            assert (d <= 1).all()
            off, total = off + int(d.sum()), total + d.numel()
        w, v = ((x["master_param"] if "master_param" in x else y.detach()).cpu().double() for x, y in ((s, p), (t, q)))
        eps = torch.finfo(torch.float32 if "master_param" in s else dtype).eps
        assert ((w - v).abs() <= (eps + 2 * 2 ** -24) * v.abs() + 16 * 2 ** -24 * lr * 40 + 2.0 ** -24 + (slack[i] if slack else 0)).all()
        if "master_param" in s:
            assert torch.equal(p.detach(), s["master_param"].to(dtype))
    assert off <= max(2, 1e-4 * total), f"{off} of {total} codes differ"


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, False), (torch.bfloat16, True), (torch.float16, True)])
@pytest.mark.parametrize("l2,bias,wd", [(False, True, 0.1), (True, False, 0.1), (False, True, 0.0)])
@pytest.mark.parametrize("capturable", [False, True])
def test_the_cpu_path(dtype, master, l2, bias, wd, capturable):
    args = dict(lr=1e-2, adam_w_mode=not l2, bias_correction=bias, weight_decay=wd, master_weights=master, seed=11)
    pa, ga = make(SIZES, dtype, device="cuda")
    pb, gb = make(SIZES, dtype)
    a, b = FusedAdam8bit(pa, capturable=capturable, **args), FusedAdam8bit(pb, **args)
    for step in range(1, 4):
        ga(step), gb(step)
        if step > 1:
            start_alike(a, b, pa, pb)
        slack = l2_slack(b, pb, 1e-2, wd) if l2 else None
        a.step(), b.step()
        same(a, b, pa, pb, 1e-2, dtype, slack)


def test_every_code_is_read_and_written():
    """State of all 127 (and with signs 253) codes passes through the kernel: with beta 1 - 2^-20 and no gradient a code's
    value all but stays, and rounds to itself or to the code below."""
    p = torch.nn.Parameter(torch.zeros(256, device="cuda"))
    opt = FusedAdam8bit([p], lr=0.0, betas=(1 - 2.0 ** -20, 1 - 2.0 ** -20), bias_correction=False)
    p.grad = torch.zeros_like(p)
    opt.step()
    st = opt.state[p]
    every = torch.arange(256, dtype=torch.uint8)
    every[127] = every[255] = 126          # NaN's places
    every[128] = 0
    for k in ("exp_avg", "exp_avg_sq"):
        x = every if k == "exp_avg" else every & 127
        st[k].copy_(x.view(torch.float8_e4m3fn).cuda())
        st[k + "_scale"].fill_(2.0)
    opt.step()
    for k in ("exp_avg", "exp_avg_sq"):
        x = (every if k == "exp_avg" else every & 127).view(torch.float8_e4m3fn).float()
        # the scale is the largest's: 2 (1 - 2^-20) or its root; then every value is its code again, to a part of 2^-20
        got = st[k].float().cpu()
        d = (got.view(torch.float32) - x).abs()
        gap = torch.maximum(x.abs() / 8, torch.tensor(2.0 ** -9))
        assert (d <= gap * 1.0001).all() and (d > 0).sum() <= 3
        torch.testing.assert_close(st[k + "_scale"].cpu(), torch.full((2,), 2.0), rtol=2.0 ** -19, atol=0)


def test_views_at_odd_addresses_and_their_neighbours():
    """Params, gradients and moments that lie end to end in one buffer; what is between and behind them stays."""
    sizes = [1, 127, 130, 5, 9000, 3]
    total = sum(sizes) + len(sizes) + 16
    def lay(dtype):
        buf = torch.full((total,), 7.0, device="cuda").to(dtype)
        views, o = [], 1
        for n in sizes:
            views.append(buf[o:o + n])
            o += n + 1
        return buf, views
    for dtype in (torch.float32, torch.bfloat16):
        bufs = [lay(dtype), lay(dtype), lay(torch.float8_e4m3fn), lay(torch.float8_e4m3fn), lay(torch.float32)]
        params = [torch.nn.Parameter(v) for v in bufs[0][1]]
        opt = FusedAdam8bit(params, lr=1e-2, master_weights=dtype != torch.float32)
        plain = [torch.nn.Parameter(v.clone()) for v in bufs[0][1]]
        opt2 = FusedAdam8bit(plain, lr=1e-2, master_weights=dtype != torch.float32)
        for i, (p, q) in enumerate(zip(params, plain)):
            p.grad = bufs[1][1][i]
            q.grad = p.grad.clone()
            st = {"exp_avg": bufs[2][1][i], "exp_avg_sq": bufs[3][1][i]}
            for k in ("exp_avg", "exp_avg_sq"):
                st[k + "_scale"] = torch.full((-(-p.numel() // BLOCK),), 0.01, device="cuda")
            if dtype != torch.float32:
                st["master_param"] = bufs[4][1][i]
            opt.state[p] = st
            opt2.state[q] = {k: v.clone() for k, v in st.items()}
        before = [b.clone() for b, _ in bufs]
        opt.step(), opt2.step()
        inside = torch.zeros(total, dtype=torch.bool, device="cuda")
        o = 1
        for n in sizes:
            inside[o:o + n] = True
            o += n + 1
        for (b, _), old in zip(bufs, before):
            assert torch.equal(b.view(torch.uint8).view(total, -1)[~inside], old.view(torch.uint8).view(total, -1)[~inside])
        for p, q in zip(params, plain):
            assert torch.equal(p, q)
            for k in opt.state[p]:
                assert torch.equal(opt.state[p][k].view(torch.uint8), opt2.state[q][k].view(torch.uint8))


def test_many_tensors_one_after_another():
    """More tensors than one launch takes, some without a gradient: the same as each kept by itself in its place."""
    sizes = [(1 + 37 * i % 300,) for i in range(150)]
    pa, ga = make(sizes, torch.float32, device="cuda")
    pb, gb = make(sizes, torch.float32)
    a, b = FusedAdam8bit(pa, lr=1e-2), FusedAdam8bit(pb, lr=1e-2)
    ga(1), gb(1)
    for i in range(0, 150, 7):
        pa[i].grad = pb[i].grad = None
    a.step(), b.step()
    for p, q in zip(pa, pb):
        assert (p in a.state) == (p.grad is not None)
    with_grad = [i for i in range(150) if pa[i].grad is not None]
    same(a, b, [pa[i] for i in with_grad], [pb[i] for i in with_grad], 1e-2, torch.float32)


def test_layouts():
    g = torch.Generator().manual_seed(5)
    w, d = torch.randn(16, 6, 5, 5, generator=g), torch.randn(16, 6, 5, 5, generator=g)
    out = []
    for grad_format in (torch.channels_last, torch.contiguous_format):
        p = torch.nn.Parameter(w.cuda().to(memory_format=torch.channels_last))
        opt = FusedAdam8bit([p], lr=1e-2)
        p.grad = d.cuda().to(memory_format=grad_format)
        opt.step()
        assert opt.state[p]["exp_avg"].stride() == p.stride()
        out.append(p.detach())
    assert torch.equal(out[0], out[1])
    q = torch.nn.Parameter(w.to(memory_format=torch.channels_last))
    opt = FusedAdam8bit([q], lr=1e-2)
    q.grad = d
    opt.step()
    torch.testing.assert_close(out[0].cpu(), q.detach(), rtol=0, atol=4 * 2 ** -24 * 5)


def test_a_tensor_beyond_32_bits():
    """2^31 + 131 elements: those behind 2^31 are stepped as a small tensor's are, but for their random numbers."""
    n, tail = 2 ** 31 + 131, 131
    g = torch.Generator().manual_seed(3)
    w, d = torch.randn(tail, generator=g), torch.randn(tail, generator=g)
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    p.detach()[-tail:] = w.cuda()
    p.grad[-tail:] = d.cuda()
    opt = FusedAdam8bit([p], lr=1e-2)
    opt.step()
    q = torch.nn.Parameter(w.bfloat16())
    q.grad = d.bfloat16()
    small = FusedAdam8bit([q], lr=1e-2)
    small.step()
    # rounded to bf16, and where fp32 differs in its last bits to the other side
    torch.testing.assert_close(p.detach()[-tail:].cpu(), q.detach(), rtol=2 ** -7, atol=0)
    for k in ("exp_avg", "exp_avg_sq"):
        s, t = opt.state[p], small.state[q]
        torch.testing.assert_close(s[k + "_scale"][-2:].cpu(), t[k + "_scale"], rtol=8 * 2 ** -24, atol=0)
        # of the two codes around a value each takes one: at most a code's distance, 1/8 of the larger or 2^-9, apart
        a, b = s[k][-tail:].cpu().float(), t[k].float()
        assert ((a - b).abs() <= torch.maximum(torch.maximum(a.abs(), b.abs()) / 8, torch.tensor(2.0 ** -9))).all()
        assert not s[k].view(torch.uint8)[:-tail].any()
    assert not p.detach()[:-tail].any()


def test_infinite_and_nan_gradients_stay_where_they_are():
    for dtype in (torch.float32, torch.bfloat16):
        p = torch.nn.Parameter(torch.ones(1000, device="cuda", dtype=dtype))
        opt = FusedAdam8bit([p], lr=1e-2)
        p.grad = torch.full_like(p, 0.5)
        p.grad[7], p.grad[200], p.grad[999] = math.inf, math.nan, -math.inf
        opt.step()
        bad = torch.zeros(1000, dtype=torch.bool)
        bad[[7, 200, 999]] = True
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(torch.isnan(opt.state[p][k].float()).cpu(), bad)
            assert torch.isfinite(opt.state[p][k + "_scale"]).all()
        assert torch.equal(torch.isfinite(p.detach().float()).cpu(), ~bad)


def test_tiny_and_huge_blocks():
    """Blocks of values whose scale would be under fp32's normal numbers, and of large ones."""
    for size in (0.0, 1e-42, 1e-38, 1e-30, 1e18):
        p, q = (torch.nn.Parameter(torch.ones(130, device=d)) for d in ("cuda", "cpu"))
        for w in (p, q):
            opt = FusedAdam8bit([w], lr=1e-2)
            w.grad = torch.full((130,), size, device=w.device)
            opt.step()
            if w is p:
                mine = opt
        s, t = mine.state[p], opt.state[q]
        for k in s:
            assert torch.isfinite(s[k].float()).all()
        torch.testing.assert_close(p.detach().cpu(), q.detach(), rtol=0, atol=16 * 2 ** -24)
        for k in ("exp_avg_scale", "exp_avg_sq_scale"):
            torch.testing.assert_close(s[k].cpu(), t[k], rtol=8 * 2 ** -24, atol=1e-37)


@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True)])
def test_captured_and_replayed(dtype, master):
    """Five replays with new gradients and a new learning rate, eager work between, each the same as an eager step."""
    pa, ga = make([(300,), (8200,)], dtype, device="cuda")
    pb, gb = make([(300,), (8200,)], dtype, device="cuda")
    a = FusedAdam8bit(pa, lr=1e-2, capturable=True, master_weights=master, weight_decay=0.1)
    b = FusedAdam8bit(pb, lr=1e-2, capturable=True, master_weights=master, weight_decay=0.1)
    ga(0), gb(0)
    a.step(), b.step()
    fixed = [p.grad for p in pa]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for step in range(1, 6):
        gb(step)
        for f, q in zip(fixed, pb):
            f.copy_(q.grad)
        if step == 3:
            a.param_groups[0]["lr"].fill_(3e-3)
            b.param_groups[0]["lr"].fill_(3e-3)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for p, q in zip(pa, pb):
            assert torch.equal(p, q)
            for k in a.state[p]:
                assert torch.equal(a.state[p][k].view(torch.uint8), b.state[q][k].view(torch.uint8))


def test_grad_scaler_skips_and_unscales():
    p = torch.nn.Parameter(torch.ones(200, device="cuda"))
    q = torch.nn.Parameter(torch.ones(200, device="cuda"))
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    a, b = FusedAdam8bit([p], lr=1e-2, capturable=True), FusedAdam8bit([q], lr=1e-2, capturable=True)
    scaler.scale(torch.zeros((), device="cuda"))
    for step in range(3):
        p.grad = torch.full_like(p, 0.25 * 1024)
        q.grad = torch.full_like(q, 0.25)
        if step == 1:
            p.grad[3] = math.inf
        before = p.detach().clone()
        scaler.step(a)
        scaler.update(1024.0)
        if step == 1:
            assert torch.equal(p, before) and int(a.param_groups[0]["step"]) == 1
        else:
            b.step()
            assert torch.equal(p, q)
    assert int(a.param_groups[0]["step"]) == 2


def test_a_checkpoint_goes_on_bit_for_bit():
    for capturable in (False, True):
        pa, ga = make([(77, 5), (300,)], torch.bfloat16, device="cuda")
        a = FusedAdam8bit(pa, lr=1e-2, master_weights=True, capturable=capturable)
        for step in range(2):
            ga(step)
            a.step()
        saved = a.state_dict()
        pb, gb = make([(77, 5), (300,)], torch.bfloat16, device="cuda")
        b = FusedAdam8bit(pb, lr=1.0, master_weights=True, capturable=capturable)
        with torch.no_grad():
            for p, q in zip(pa, pb):
                q.copy_(p)
        b.load_state_dict(saved)
        for step in range(2, 4):
            ga(step), gb(step)
            a.step(), b.step()
        for p, q in zip(pa, pb):
            assert torch.equal(p, q) and torch.equal(a.state[p]["master_param"], b.state[q]["master_param"])
            assert a.state[p]["exp_avg"].data_ptr() != b.state[q]["exp_avg"].data_ptr()


def test_a_side_stream():
    pa, ga = make([(5000,)], torch.float32, device="cuda")
    pb, gb = make([(5000,)], torch.float32, device="cuda")
    ga(1), gb(1)
    a, b = FusedAdam8bit(pa), FusedAdam8bit(pb)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    b.step()
    torch.cuda.synchronize()
    assert torch.equal(pa[0], pb[0])


def test_a_post_training_step_of_all_of_them():
    """A small decoder is held near its frozen copy: the copy's log-probabilities, a policy and a preference step with
    the gradients of the formulas in plain torch, and the optimizer over them."""
    from apex_amd.contrib.xentropy import policy_loss, preference_loss, sequence_log_probs, token_log_probs
    from apex_amd.models.transformer import LlamaModel, TransformerLMConfig

    torch.manual_seed(0)
    cfg = TransformerLMConfig(vocab_size=211, hidden=128, layers=2, heads=2, seq_len=32, ffn_hidden=192, causal=True, norm="rmsnorm")
    model, frozen = LlamaModel(cfg).cuda().bfloat16(), LlamaModel(cfg).cuda().bfloat16()
    frozen.load_state_dict(model.state_dict())
    opt = FusedAdam8bit(model.parameters(), lr=1e-3, master_weights=True, weight_decay=0.01)
    tokens = torch.randint(0, 211, (4, 32), device="cuda")
    labels = torch.cat([tokens[:, 1:], torch.full((4, 1), -100, device="cuda")], 1)
    labels[:, :8] = -100
    on = labels != -100
    with torch.no_grad():
        x = frozen(tokens)
        old, ref = token_log_probs(x, labels), sequence_log_probs(x, labels)
        # 23 tokens' fp32 sums of values of about 6
        torch.testing.assert_close(old.sum(-1), ref, rtol=0, atol=24 * 2 ** -24 * 23 * 8)
    for step in range(3):
        for kind in ("policy", "preference"):
            logits = model(tokens)
            mine = logits.detach().requires_grad_(True)
            plain = logits.detach().double().requires_grad_(True)
            lp = torch.log_softmax(plain, -1).gather(-1, labels.clamp(min=0).unsqueeze(-1)).squeeze(-1)
            if kind == "policy":
                adv = torch.tensor([1.0, -1.0, 0.5, -0.5], device="cuda")
                loss, _ = policy_loss(mine, labels, old, adv, ref_log_probs=old, kl_coef=0.1, grad_scale=1.0)
                r, a = torch.exp(lp - old), adv[:, None]
                want = (-torch.minimum(r * a, r.clamp(0.8, 1.2) * a) + 0.1 * (torch.exp(old - lp) - (old - lp) - 1))[on].mean()
            else:
                loss, chosen, _ = preference_loss(mine, labels, ref, beta=0.1)
                gain = torch.where(on, lp, 0.0).sum(-1) - ref
                want = -torch.nn.functional.logsigmoid(0.1 * (gain[:2] - gain[2:])).mean()
                assert chosen.shape == (2,)
            g, w = torch.autograd.grad(loss, mine)[0], torch.autograd.grad(want, plain)[0]
            torch.testing.assert_close(loss.double(), want, rtol=0, atol=1e-4)
            # one rounding to bf16 and fp32's part of a size of 1 / 92 (policy) or beta / 2 (preference)
            torch.testing.assert_close(g.double(), w, rtol=2 ** -8 * 1.01, atol=1e-5)
            assert (g[~on] == 0).all()
            opt.zero_grad()
            logits.backward(g)
            before = [p.detach().clone() for p in model.parameters()]
            opt.step()
            for p, b in zip(model.parameters(), before):
                assert torch.isfinite(p).all() and (p.numel() < 1000 or not torch.equal(p, b))


@pytest.mark.parametrize("level", ["O1", "O2"])
def test_under_amp(level):
    """amp's own masters (O2) and its loss scale. The first step is FusedAdam's, for it is made of moments that have not
    been rounded yet: weights under 1 and a step of lr differ by some half steps of fp32. Later steps go on."""
    from apex_amd import amp
    from apex_amd.optimizers import FusedAdam

    first = []
    for cls in (FusedAdam8bit, FusedAdam):
        torch.manual_seed(0)
        net = torch.nn.Sequential(torch.nn.Linear(64, 200), torch.nn.ReLU(), torch.nn.Linear(200, 8)).cuda()
        opt = cls(net.parameters(), lr=1e-2)
        net, opt = amp.initialize(net, opt, opt_level=level, cast_model_type=torch.bfloat16, loss_scale=128.0, verbosity=0)
        x = torch.randn(32, 64, device="cuda")
        for step in range(3):
            before = [p.detach().clone() for p in amp.master_params(opt)]
            loss = net(x).float().square().mean()
            with amp.scale_loss(loss, opt) as scaled:
                scaled.backward()
            opt.step()
            opt.zero_grad()
            after = [p.detach().clone() for p in amp.master_params(opt)]
            assert all(torch.isfinite(p).all() and not torch.equal(p, b) for p, b in zip(after, before))
            if step == 0:
                first.append(after)
    for a, b in zip(*first):
        # FusedAdam takes 1 - beta2 in fp32, which is 1.3e-5 off, and so is half of it in a step; a weight that is held in
        # 16 bits may be rounded to the other side
        assert a.dtype == (torch.float32 if level == "O2" else torch.bfloat16)
        torch.testing.assert_close(a, b, rtol=torch.finfo(a.dtype).eps + 4 * 2 ** -24, atol=1e-2 * (1.3e-5 + 32 * 2 ** -24))


@pytest.mark.parametrize("unscale", [False, True])
def test_a_scaler_that_has_unscaled_already(unscale):
    """unscale_, clip, step: the step is that of the true gradients, bit for bit (the scale is a power of two), at an eps
    that tells their size; one that is not finite skips it and does not count."""
    sizes = [(3, 50), (129,), (5000,)]
    pa, _ = make(sizes, torch.float32, device="cuda")
    pb, gb = make(sizes, torch.float32, device="cuda")
    a, b = (FusedAdam8bit([{"params": p[:1]}, {"params": p[1:]}], lr=1e-2, eps=1e-2, capturable=True) for p in (pa, pb))
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0, growth_interval=1000)
    scaler.scale(torch.zeros((), device="cuda"))
    for step in range(3):
        gb(step)
        for p, q in zip(pa, pb):
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
        else:
            b.step()
        assert [int(x["step"]) for x in a.param_groups] == [(1, 1, 2)[step]] * 2
        for p, q in zip(pa, pb):
            assert torch.equal(p, q)
            for k in a.state[p]:
                assert torch.equal(a.state[p][k].view(torch.uint8), b.state[q][k].view(torch.uint8))


def test_what_one_device_found_holds_for_all():
    """Params on the GPU and on the CPU: a gradient on either that is not finite skips both."""
    p, q = (torch.nn.Parameter(torch.ones(200, device=d)) for d in ("cuda", "cpu"))
    opt = FusedAdam8bit([{"params": [p]}, {"params": [q]}], lr=1e-2, capturable=True)
    scaler = torch.amp.GradScaler("cuda", init_scale=64.0, growth_interval=1000)
    scaler.scale(torch.zeros((), device="cuda"))
    for bad in (p, q, None):
        for w in (p, q):
            w.grad = torch.full_like(w, 64.0 * 0.25)
        if bad is not None:
            bad.grad[3] = math.inf
        scaler.step(opt)
        scaler.update(64.0)
        for w in (p, q):
            assert torch.equal(w.detach(), torch.ones_like(w)) == (bad is not None)
    assert [int(g["step"]) for g in opt.param_groups] == [1, 1]
    torch.testing.assert_close(p.detach().cpu(), q.detach(), rtol=0, atol=4 * 2 ** -24)


@pytest.mark.parametrize("size", [2e-21, 1e-20, 1e-19, 1e-18, 3e-18, 1e-17, 1e-14, 1e19, 5.8e20, 7e20, 1e30, 3e38])
def test_the_root_at_both_ends(size):
    """Second moments that are subnormal or just over it (gradients up to some 1e-17), close to fp32's largest (5.8e20)
    and infinite (from 5.83e20 on: their code is NaN, and the step is m / inf = 0), beside gradients of 0. v and m are the
    same operations on both sides; the root, the quotient and the products are off by under 16 half steps together."""
    g = size * (1 + torch.rand(300, generator=torch.Generator().manual_seed(0)) / 64)
    g[::7] = 0
    g.clamp_(max=torch.finfo(torch.float32).max)
    out = []
    for device in ("cuda", "cpu"):
        p = torch.nn.Parameter(torch.zeros(300, device=device))
        opt = FusedAdam8bit([p], lr=1e-2, eps=1e-30, bias_correction=False)
        p.grad = g.to(device)
        opt.step()
        out.append((p.detach().cpu(), {k: v.cpu() for k, v in opt.state[p].items()}))
    (p, s), (q, t) = out
    torch.testing.assert_close(p, q, rtol=16 * 2 ** -24, atol=0)
    over = (torch.tensor(1 - 0.999, dtype=torch.float32) * g * g).isinf()
    assert torch.equal(t["exp_avg_sq"].float().isnan(), over) and torch.equal(p == 0, over | (g == 0))
    for k in ("exp_avg", "exp_avg_sq"):
        torch.testing.assert_close(s[k + "_scale"], t[k + "_scale"], rtol=8 * 2 ** -24, atol=0)
        # a code by one where a value lies within those half steps of its threshold: hardly ever
        a, b = s[k].float(), t[k].float()
        assert torch.equal(a.isnan(), b.isnan()) and (a.nan_to_num() != b.nan_to_num()).sum() <= 2


def test_masters_after_a_checkpoint_without_them():
    """Made in the first eager step, and the step is the CPU path's; a capture that would make them is refused."""
    pa, ga = make([(300,), (77, 5)], torch.bfloat16, device="cuda")
    a = FusedAdam8bit(pa, lr=1e-2, capturable=True)
    ga(0)
    a.step()
    for capture in (True, False):
        pb, gb = make([(300,), (77, 5)], torch.bfloat16, device="cuda")
        b = FusedAdam8bit(pb, lr=1e-2, capturable=True, master_weights=True)
        b.load_state_dict(a.state_dict())
        gb(1)
        if not capture:
            b.step()
            continue
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="before capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                b.step()
    pc, gc = make([(300,), (77, 5)], torch.bfloat16)
    c = FusedAdam8bit(pc, lr=1e-2, master_weights=True)
    c.load_state_dict(a.state_dict())
    gc(1)
    c.step()
    same(b, c, pb, pc, 1e-2, torch.bfloat16)
    assert all(torch.equal(p.detach(), b.state[p]["master_param"].bfloat16()) for p in pb)


def test_a_first_step_is_not_captured():
    """Its state would be made anew, with moments of 0 and step 1, at every replay: refused, also where only one param
    meets its first gradient, and what was there stays."""
    pa, ga = make([(300,), (77, 5)], torch.float32, device="cuda")
    opt = FusedAdam8bit(pa, lr=1e-2, capturable=True)
    for taken in (False, True):
        ga(0)
        if taken:
            pa[1].grad = None
            opt.step()
            ga(1)
        before = [p.detach().clone() for p in pa]
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="before capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, b) for p, b in zip(pa, before))
    opt.step()
    assert len(opt.state) == 2 and int(opt.param_groups[0]["step"]) == 2


def test_a_capture_needs_capturable():
    """Without it step, lr and the random numbers of the rounding would be the captured step's for ever."""
    pa, ga = make([(300,)], torch.float32, device="cuda")
    opt = FusedAdam8bit(pa, lr=1e-2)
    ga(0)
    opt.step()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="capturable=True"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    assert opt.param_groups[0]["step"] == 1
    opt.step()


def test_a_refused_step_changes_nothing():
    """A tensor that does not fit, behind those of a first launch: found before any is stepped."""
    pa, ga = make([(10,)] * 60, torch.float32, device="cuda")
    opt = FusedAdam8bit(pa, lr=1e-2)
    ga(0)
    opt.step()
    good = opt.state[pa[55]]["exp_avg_scale"]
    opt.state[pa[55]]["exp_avg_scale"] = torch.zeros(5, device="cuda")
    before = [p.detach().clone() for p in pa] + [opt.state[p]["exp_avg"].clone() for p in pa]
    with pytest.raises(RuntimeError, match="size mismatch"):
        opt.step()
    for b, a in zip(before, pa + [opt.state[p]["exp_avg"] for p in pa]):
        assert torch.equal(b.view(torch.uint8), a.detach().view(torch.uint8))
    opt.state[pa[55]]["exp_avg_scale"] = good
    opt.step()


def test_more_elements_than_one_grid_has_threads_for():
    """9 params of 2^31 elements: 2^34 and more, four a thread. The first step is lr everywhere (m over the root of v is 1),
    and a moment is the same code for every element: each is its block's largest."""
    n = 2 ** 31
    grad = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    params = [torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda")) for _ in range(9)]
    for p in params:
        p.grad = grad
    opt = FusedAdam8bit(params, lr=2.0 ** -7)
    opt.step()
    for p in params:
        # a step of 2^-7 (1 - 2 half steps and eps / 0.5) is 2^-7 in bf16
        assert p.detach().min() == p.detach().max() == -(2.0 ** -7)
        for k in ("exp_avg", "exp_avg_sq"):
            top = opt.state[p][k].view(torch.uint8)
            assert top.min() == top.max() == 126
            scale = opt.state[p][k + "_scale"]
            assert scale.min() == scale.max() > 0
    del params, opt, grad, p, top, scale
    torch.cuda.empty_cache()
