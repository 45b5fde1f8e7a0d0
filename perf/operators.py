"""The operators of a post-training step, as a program calls them, on sizes that such programs have.

Four operators that meet in one step: per-token log-probabilities (a frozen reference scores the batch with
them), the preference loss over pairs of answers, the clipped policy loss with its KL term, and an Adam step
whose two moments are held in 8 bits, so that the reference model fits beside the policy.

Where ``own`` is false, ``run`` computes each in plain torch operations in 32 bits. Where it is true, ``run``
calls apex_amd. ``exact`` computes the same from the definitions in 64 bits.
"""

import math

import torch

own = False

IGNORE = -100
BLOCK = 128  # elements of a tensor that share one scale of an 8-bit moment
TOP = 448.0  # the largest e4m3 value
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- the cases -------------------------------------------------------------------------------------------------


def listed():
    return [
        # eight candidate continuations scored for their next token: latency
        dict(name="tokens one each", op="tokens", seqs=8, length=1, vocab=50304, dtype="bf16", backward=False, temperature=1.0),
        # a frozen reference scores a batch of answers; prompts and padding are ignored
        dict(name="tokens reference", op="tokens", seqs=8, length=1024, vocab=32000, dtype="bf16", backward=False, temperature=1.0),
        # fine-tuning on weighted tokens in full precision, an odd vocabulary, sampled at a temperature
        dict(name="tokens weighted", op="tokens", seqs=4, length=777, vocab=50257, dtype="fp32", backward=True, temperature=0.7),
        # two pairs of short answers in fp16, with columns that pad the vocabulary
        dict(name="pairs short", op="pairs", pairs=2, length=128, vocab=30528, banned=6, dtype="fp16", packed=False, kind="sigmoid", average=False, smoothing=0.0),
        # a padded batch of eight pairs
        dict(name="pairs padded", op="pairs", pairs=8, length=1024, vocab=32000, banned=0, dtype="bf16", packed=False, kind="sigmoid", average=False, smoothing=0.1),
        # pairs of ragged answers laid end to end, length-averaged, squared loss
        dict(name="pairs packed", op="pairs", pairs=11, length=509, vocab=50257, banned=0, dtype="bf16", packed=True, kind="ipo", average=True, smoothing=0.0),
        # a group of eight short answers to one prompt
        dict(name="policy group", op="policy", seqs=8, length=96, vocab=32000, dtype="bf16", kl=0.04, high=0.28, reduction="sequence", temperature=1.0, at_once=False),
        # a step of many long answers
        dict(name="policy step", op="policy", seqs=16, length=2048, vocab=50304, dtype="bf16", kl=0.01, high=0.2, reduction="token", temperature=1.0, at_once=False),
        # a large vocabulary, the gradient made in the pass that reads the logits
        dict(name="policy at once", op="policy", seqs=4, length=1024, vocab=131072, dtype="bf16", kl=0.0, high=0.2, reduction="token", temperature=0.9, at_once=True),
        # adapters and norms of a small model: launches count
        dict(name="adam small", op="adam", layers=4, hidden=65, ffn=173, vocab=257, dtype="fp32", master=False, align=1),
        # a decoder's weights in bf16 with 32-bit master copies
        dict(name="adam master", op="adam", layers=12, hidden=2048, ffn=5632, vocab=32000, dtype="bf16", master=True, align=128),
        # a decoder's weights in 32 bits
        dict(name="adam fp32", op="adam", layers=6, hidden=1536, ffn=4100, vocab=30011, dtype="fp32", master=False, align=4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tokens", "pairs", "policy", "adam"])
    if op == "adam":
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        hidden = _log(rng, 33, 2048)
        return dict(op=op, layers=rng.randint(1, 10), hidden=hidden, ffn=int(hidden * rng.uniform(1.5, 2.75)), vocab=_log(rng, 100, 32000),
                    dtype=dtype, master=dtype != "fp32", align=rng.choice([1, 4, 128]))
    vocab = _log(rng, 1000, 131072)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    most = (1 << 30) // (vocab * (2 if dtype == "fp32" else 1))
    rows = _log(rng, 16, min(32768, most))
    if op == "tokens":
        seqs = rng.randint(1, 16)
        return dict(op=op, seqs=seqs, length=max(1, rows // seqs), vocab=vocab, dtype=dtype, backward=rng.random() < 0.6, temperature=round(rng.uniform(0.5, 1.5), 3))
    if op == "pairs":
        pairs = rng.randint(1, 12)
        return dict(op=op, pairs=pairs, length=max(4, rows // (2 * pairs)), vocab=vocab, banned=rng.choice([0, 1, 47]), dtype=dtype, packed=rng.random() < 0.5,
                    kind=rng.choice(["sigmoid", "ipo", "hinge"]), average=rng.random() < 0.5, smoothing=0.0)
    seqs = rng.randint(1, 16)
    return dict(op=op, seqs=seqs, length=max(4, rows // seqs), vocab=vocab, dtype=dtype, kl=rng.choice([0.0, 0.05]), high=rng.choice([0.2, 0.3]),
                reduction=rng.choice(["token", "sequence"]), temperature=round(rng.uniform(0.7, 1.2), 3), at_once=rng.random() < 0.5)


def _spans(case):
    """(first answer token, end) of each sequence, and its length as laid out: prompts come first, padding last."""
    n = 2 * case["pairs"] if case["op"] == "pairs" else case["seqs"]
    length, spans = case["length"], []
    if length < 4:
        return [(0, length)] * n
    for i in range(n):
        end = length - (i * 37 + 11) % (length // 4 + 1)
        spans.append((min(end - 1, length * (1 + i % 4) // 8), end))
    return spans


def _rows(case):
    """All rows of the logits, and those of an answer's tokens."""
    spans = _spans(case)
    every = sum(e for _, e in spans) if case.get("packed") else len(spans) * case["length"]
    return every, sum(e - b for b, e in spans)


def _shapes(case):
    h, f = case["hidden"], case["ffn"]
    layer = [(3 * h, h), (h, h), (f, h), (f, h), (h, f), (h,), (h,)]
    return [(case["vocab"], h)] + layer * case["layers"] + [(h,)]


def work(case):
    if case["op"] == "adam":
        n = sum(math.prod(s) for s in _shapes(case))
        blocks = sum(-(-math.prod(s) // BLOCK) for s in _shapes(case))
        size = TYPES[case["dtype"]].itemsize
        # gradient in, weights and both moments in and out, and the master copy; a master copy spares reading the weights
        each = (2 * size + 8 if case["master"] else 3 * size) + 4
        return {"bytes": n * each + 16 * blocks, "flops": 20 * n}
    rows, answers = _rows(case)
    size = case["vocab"] * TYPES[case["dtype"]].itemsize
    back = case["op"] != "tokens" or case["backward"]
    small = 12 + (12 if case["op"] == "policy" else 0)  # labels, log-probabilities, and what the policy loss has for each token
    return {"bytes": answers * size + (rows * size if back else 0) + rows * small, "flops": answers * case["vocab"] * (8 if back else 4)}


# ---- inputs ----------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_adam(case, seed, g) if case["op"] == "adam" else _prepare_loss(case, g)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _prepare_loss(case, g):
    spans, vocab = _spans(case), case["vocab"]
    packed = case.get("packed", False)
    rows, _ = _rows(case)
    lead = (rows,) if packed else (len(spans), case["length"])
    logits = _randn(g, *lead, vocab, dtype=TYPES[case["dtype"]]).mul_(2.5)
    if case.get("banned"):
        logits[..., vocab - case["banned"]:] = -math.inf
    where = torch.zeros(rows, dtype=torch.bool, device="cuda")
    starts = [0]
    for i, (begin, end) in enumerate(spans):
        at = starts[-1] if packed else i * case["length"]
        where[at + begin: at + end] = True
        starts.append(starts[-1] + end)
    labels = torch.randint(0, vocab - case.get("banned", 0), (rows,), generator=g, device="cuda")
    # answers were sampled from a model near this one: their tokens stand high
    flat = logits.view(rows, vocab)
    flat[torch.arange(rows, device="cuda"), labels] = (_randn(g, rows) * 2 + 10).to(flat.dtype)
    labels = torch.where(where, labels, IGNORE).view(lead)
    s = {"case": case, "logits": logits, "labels": labels}
    if packed:
        s["cu_seqlens"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case["op"] == "tokens":
        s["weights"] = _randn(g, *lead)
    else:
        s["scale"] = torch.tensor(_scale(case), device="cuda")
        near = torch.cat([_near(x, y, case.get("temperature", 1.0)) for x, y in zip(flat.split(2048), labels.view(-1).split(2048))])
        moved = 0.15 * _randn(g, rows)
        if case["op"] == "pairs":  # a policy on its way: each answer has become likelier or less so than it was
            moved = moved + 0.05 * _randn(g, len(spans))[_sequence_of(s, labels)]
        if case["op"] == "policy":  # no ratio so near a clip's border that 32 bits cannot tell its side
            for border in (1 - 0.2, 1 + case["high"]):
                moved = torch.where((moved + math.log(border)).abs() < 1e-3, 0.0, moved)
        near = near + moved
        if case["op"] == "pairs":
            near = torch.where(where, near, 0.0).double()
            sums = [near[a:b].sum() for a, b in (zip(starts, starts[1:]) if packed else ((i * case["length"], (i + 1) * case["length"]) for i in range(len(spans))))]
            ref = torch.stack(sums)
            if case["average"]:
                ref = ref / torch.tensor([e - b for b, e in spans], device="cuda")
            s["ref"] = ref.float()
        else:
            s["old"] = near.view(lead)
            s["ref"] = (near + 0.3 * _randn(g, rows)).view(lead) if case["kl"] else None
            s["advantages"] = _randn(g, len(spans)) + 0.25
    if case["op"] != "tokens" or case["backward"]:
        logits.requires_grad_(True)
    return s


def _scale(case):
    """What the loss is multiplied by before its backward pass: gradients of one token in thousands are too small for fp16."""
    return 16384.0 if case["dtype"] == "fp16" else 1.0


def _near(x, y, temperature):
    x = x.float() / temperature
    return x.gather(-1, y.clamp(min=0).unsqueeze(-1)).squeeze(-1) - torch.logsumexp(x, -1)


def _prepare_adam(case, seed, g):
    shapes, dtype = _shapes(case), TYPES[case["dtype"]]
    sizes = [math.prod(s) for s in shapes]
    at, block, places = 0, 0, []
    for n in sizes:
        places.append((at, block, n))
        at += -(-n // case["align"]) * case["align"]
        block += -(-n // BLOCK)
    weights = _randn(g, at) * 0.02
    s = {"case": case, "shapes": shapes, "places": places, "seed": seed % 10007, "step": 100 + seed % 50, "group": dict(lr=2e-5, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)}
    s["param"] = weights.to(dtype)
    s["master"] = weights if case["master"] else None
    spread = torch.exp(0.7 * _randn(g, at))  # some weights have larger gradients than others
    s["grad"] = (1e-3 * spread * _randn(g, at)).to(dtype)
    m, r = 3e-4 * spread * _randn(g, at), 1e-3 * spread * (0.3 + torch.rand(at, generator=g, device="cuda"))
    for name, x in (("exp_avg", m), ("exp_avg_sq", r)):
        codes = torch.zeros(at, dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty(block, device="cuda")
        for o, b, n in places:
            rows = _in_blocks(x[o: o + n])
            scale = rows.abs().amax(1) / TOP
            codes[o: o + n] = (rows / scale[:, None]).to(torch.float8_e4m3fn).view(-1)[:n]
            scales[b: b + rows.shape[0]] = scale
        s[name], s[name + "_scale"] = codes, scales
    if own:
        s["optimizer"] = _optimizer(s)
    return s


def _in_blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _optimizer(s):
    """The optimizer of a run that is under way: its moments are what a checkpoint would have put there."""
    from apex_amd.optimizers import FusedAdam8bit

    params = []
    for (o, _, n), shape in zip(s["places"], s["shapes"]):
        p = torch.nn.Parameter(s["param"][o: o + n].view(shape))
        p.grad = s["grad"][o: o + n].view(shape)
        params.append(p)
    opt = FusedAdam8bit(params, master_weights=s["master"] is not None, seed=s["seed"], **s["group"])
    for p, (o, b, n), shape in zip(params, s["places"], s["shapes"]):
        state = {k: s[k][o: o + n].view(shape) for k in ("exp_avg", "exp_avg_sq")}
        state |= {k + "_scale": s[k + "_scale"][b: b - (-n // BLOCK)] for k in ("exp_avg", "exp_avg_sq")}
        if s["master"] is not None:
            state["master_param"] = s["master"][o: o + n].view(shape)
        opt.state[p] = state
    opt.param_groups[0]["step"] = s["step"]
    return opt


# ---- one pass --------------------------------------------------------------------------------------------------


def run(state):
    return {"tokens": _tokens, "pairs": _pairs, "policy": _policy, "adam": _adam}[state["case"]["op"]](state)


def _tokens(s):
    case, x, y = s["case"], s["logits"], s["labels"]
    if own:
        from apex_amd.contrib.xentropy import token_log_probs

        lp = token_log_probs(x, y, temperature=case["temperature"])
        return [lp, torch.autograd.grad(lp, x, s["weights"])[0]] if case["backward"] else [lp]
    lp, p = _plain_log_probs(x.detach(), y, case["temperature"])
    return [lp, _plain_gradient(p, y, s["weights"], case["temperature"], x.dtype)] if case["backward"] else [lp]


def _pairs(s):
    case, x, y = s["case"], s["logits"], s["labels"]
    if own:
        from apex_amd.contrib.xentropy import preference_loss

        loss, chosen, rejected = preference_loss(x, y, s["ref"], beta=0.1, label_smoothing=case["smoothing"], loss_type=case["kind"],
                                                 average=case["average"], cu_seqlens=s.get("cu_seqlens"))
        return [loss.detach(), chosen, rejected, torch.autograd.grad(loss, x, s["scale"])[0]]
    beta, eps = 0.1, case["smoothing"]
    lp, p = _plain_log_probs(x.detach(), y, 1.0, wide=torch.float64)  # tokens are added up: no error that they share
    which = _sequence_of(s, y)
    n = 2 * case["pairs"]
    active = (y != IGNORE).view(-1)
    sums = torch.zeros(n, dtype=torch.float64, device="cuda").index_add_(0, which, lp.view(-1))
    count = torch.zeros(n, dtype=torch.float64, device="cuda").index_add_(0, which, active.double()).clamp(min=1) if case["average"] else torch.ones(n, dtype=torch.float64, device="cuda")
    gain = sums / count - s["ref"].double()
    chosen, rejected = gain.chunk(2)
    d = chosen - rejected
    if case["kind"] == "sigmoid":
        loss = (1 - eps) * torch.log1p(torch.exp(-beta * d)) + eps * torch.log1p(torch.exp(beta * d))
        slope = -beta * (1 - eps) / (1 + torch.exp(beta * d)) + beta * eps / (1 + torch.exp(-beta * d))
    elif case["kind"] == "ipo":
        loss = (d - 1 / (2 * beta)) ** 2
        slope = 2 * (d - 1 / (2 * beta))
    else:
        loss = (1 - beta * d).clamp(min=0)
        slope = torch.where(beta * d < 1, -beta, 0.0)
    coef = torch.cat([slope, -slope]) / (case["pairs"] * count)
    grad = _plain_gradient(p, y, (s["scale"] * coef[which]).view(y.shape).float(), 1.0, x.dtype)
    return [loss.mean().float(), (beta * chosen).float(), (beta * rejected).float(), grad]


def _policy(s):
    case, x, y = s["case"], s["logits"], s["labels"]
    if own:
        from apex_amd.contrib.xentropy import policy_loss

        loss, lp = policy_loss(x, y, s["old"], s["advantages"], ref_log_probs=s["ref"], clip_eps=0.2, clip_eps_high=case["high"], kl_coef=case["kl"],
                               temperature=case["temperature"], reduction=case["reduction"], grad_scale=_scale(case) if case["at_once"] else None)
        return [loss.detach(), lp, torch.autograd.grad(loss, x, s["scale"])[0]]
    lp, p = _plain_log_probs(x.detach(), y, case["temperature"])
    active = y != IGNORE
    a = s["advantages"][:, None]
    ratio = torch.exp(torch.where(active, lp - s["old"], 0.0))
    held = ratio.clamp(1 - 0.2, 1 + case["high"])
    each = -torch.minimum(ratio * a, held * a)
    slope = torch.where(ratio * a <= held * a, -ratio * a, 0.0)
    if s["ref"] is not None:
        d = torch.where(active, s["ref"] - lp, 0.0)
        each = each + case["kl"] * (torch.exp(d) - d - 1)
        slope = slope + case["kl"] * (1 - torch.exp(d))
    weight = active.float() / (active.sum() if case["reduction"] == "token" else active.sum(1, keepdim=True).clamp(min=1) * y.shape[0])
    loss = (each.double() * weight.double()).sum().float()
    return [loss, lp, _plain_gradient(p, y, s["scale"] * slope * weight, case["temperature"], x.dtype)]


def _sequence_of(s, y):
    if "cu_seqlens" in s:
        return torch.bucketize(torch.arange(y.numel(), device="cuda"), s["cu_seqlens"][1:].long(), right=True)
    return torch.arange(y.numel(), device="cuda") // y.shape[1]


def _plain_log_probs(x, y, temperature, wide=torch.float32):
    """The labels' log-probabilities (0 where there is no label) and all probabilities."""
    x = x.float() / temperature
    picked = x.gather(-1, y.clamp(min=0).unsqueeze(-1))
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True, dtype=wide)
    lp = (picked.to(wide) - top - torch.log(total)).squeeze(-1)
    return torch.where(y != IGNORE, lp, 0.0), e.div_(total.float())


def _plain_gradient(p, y, coef, temperature, dtype):
    """The logits' gradient, where `coef` is that of the labels' log-probabilities: coef * (1[label] - p) / temperature."""
    coef = (torch.where(y != IGNORE, coef, 0.0) / temperature).unsqueeze(-1)
    g = p.mul_(-coef)
    return g.scatter_add_(-1, y.clamp(min=0).unsqueeze(-1), coef).to(dtype)


# ---- Adam with moments in 8 bits -------------------------------------------------------------------------------
# A block of 128 elements has one scale s = max|x| / 448 and codes q in e4m3, x = s q. The first moment is held as
# it is, the second as its root. A value between two codes becomes one of them at random, so that a slow average
# moves at all: with the odds that keep the mean of the first moment, and of the second (not of its root). A second
# moment over zero stays over zero. Element i of tensor t takes two 16-bit numbers from a 32-bit hash of
# (seed, step, t, i): the low half for the first moment, the high half for the second.

MASK = 0xFFFFFFFF


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK
    return x ^ (x >> 16)


def _bits(seed, step, tensor, n):
    key = _mix((seed & MASK) ^ _mix((step + _mix((tensor + 0x6A09E667) & MASK)) & MASK))
    return _mix((torch.arange(n, device="cuda") * 0x9E3779B1 + key) & MASK)


def _adam(s):
    names = ("param", "master", "exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
    if own:
        s["optimizer"].step()
    else:
        s["step"] += 1
        [_plain_adam(s, t, *place) for t, place in enumerate(s["places"])]
    return [s[k] for k in names if s[k] is not None]


def _plain_adam(s, t, o, b, n):
    group = s["group"]
    (b1, b2), lr, wd, eps = group["betas"], group["lr"], group["weight_decay"], group["eps"]
    part, blocks = slice(o, o + n), slice(b, b - (-n // BLOCK))
    bits = _bits(s["seed"], s["step"], t, n)
    g = s["grad"][part].float()
    p = (s["param"] if s["master"] is None else s["master"])[part].float()
    m = b1 * (_in_blocks(s["exp_avg"][part].float()) * s["exp_avg_scale"][blocks, None]).view(-1)[:n] + (1 - b1) * g
    r = (_in_blocks(s["exp_avg_sq"][part].float()) * s["exp_avg_sq_scale"][blocks, None]).view(-1)[:n]
    v = b2 * r * r + (1 - b2) * g * g
    r = torch.sqrt(v)
    update = m / (1 - b1 ** s["step"]) / (r / math.sqrt(1 - b2 ** s["step"]) + eps) + wd * p
    p = p - lr * update
    s["param"][part] = p.to(s["param"].dtype)
    if s["master"] is not None:
        s["master"][part] = p
    s["exp_avg"][part], s["exp_avg_scale"][blocks] = _plain_codes(m, ((bits & 0xFFFF).float() + 0.5) / 65536, False)
    s["exp_avg_sq"][part], s["exp_avg_sq_scale"][blocks] = _plain_codes(r, ((bits >> 16).float() + 0.5) / 65536, True)


def _plain_codes(x, u, root):
    n, rows = x.numel(), _in_blocks(x)
    scale = (rows.abs().amax(1) / TOP).clamp(min=2.0 ** -126)
    y = (rows * (1 / scale)[:, None]).view(-1)[:n]
    size = y.abs().clamp(max=TOP)
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=2.0 ** -6))) - 3)
    z = size / step
    k = torch.floor(z)
    up = u * (2 * k + 1) < (z - k) * (z + k) if root else u < z - k
    k = k + up
    if root:
        k = torch.where((x > 0) & (k < 1), 1.0, k)
    return (torch.sign(y) * k * step).to(torch.float8_e4m3fn), scale


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _exact_adam(s) if case["op"] == "adam" else _exact_loss(s)


def _exact_loss(s):
    case, y = s["case"], s["labels"].reshape(-1)
    rows = y.numel()
    x = s["logits"].detach().view(rows, -1)
    t = case.get("temperature", 1.0)
    lp = torch.zeros(rows, dtype=torch.float64, device="cuda")
    active = y != IGNORE
    for i in range(0, rows, 1024):
        z = torch.log_softmax(x[i: i + 1024].double() / t, -1)
        lp[i: i + 1024] = z[torch.arange(z.shape[0], device="cuda"), y[i: i + 1024].clamp(min=0)]
    lp = torch.where(active, lp, torch.zeros_like(lp)).requires_grad_(True)
    if case["op"] == "tokens":
        outs, coef = [lp.detach().view(s["labels"].shape)], s["weights"].double().view(-1)
        if not case["backward"]:
            return outs
    elif case["op"] == "pairs":
        if case["packed"]:
            cu = s["cu_seqlens"].tolist()
        else:
            cu = list(range(0, rows + 1, case["length"]))
        total = torch.stack([lp[a:b].sum() / (max(1, int(active[a:b].sum())) if case["average"] else 1) for a, b in zip(cu, cu[1:])])
        gain = 0.1 * (total - s["ref"].double())
        c, r = gain[: case["pairs"]], gain[case["pairs"]:]
        if case["kind"] == "sigmoid":
            f = torch.nn.functional.softplus
            loss = ((1 - case["smoothing"]) * f(r - c) + case["smoothing"] * f(c - r)).mean()
        elif case["kind"] == "ipo":
            loss = ((c - r) / 0.1 - 5.0).square().mean()
        else:
            loss = torch.relu(1 - (c - r)).mean()
        outs = [loss.detach(), c.detach(), r.detach()]
        coef = _scale(case) * torch.autograd.grad(loss, lp)[0]
    else:
        a = s["advantages"].double().repeat_interleave(case["length"])
        ratio = (lp - s["old"].double().view(-1)).exp()
        each = torch.maximum(-a * ratio, -a * ratio.clamp(0.8, 1 + case["high"]))
        if s["ref"] is not None:
            d = s["ref"].double().view(-1) - lp
            each = each + case["kl"] * (torch.expm1(d) - d)
        if case["reduction"] == "token":
            loss = each[active].mean()
        else:
            loss = torch.stack([e[k].mean() for e, k in zip(each.view(s["labels"].shape), active.view(s["labels"].shape))]).mean()
        outs = [loss.detach(), lp.detach().view(s["labels"].shape)]
        coef = _scale(case) * torch.autograd.grad(loss, lp)[0]
    coef = torch.where(active, coef, torch.zeros_like(coef)) / t
    grad = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for i in range(0, rows, 1024):
        p = torch.softmax(x[i: i + 1024].double() / t, -1)
        p[torch.arange(p.shape[0], device="cuda"), y[i: i + 1024].clamp(min=0)] -= 1
        grad[i: i + 1024] = -coef[i: i + 1024, None] * p
    return outs + [grad.view(s["logits"].shape)]


def _exact_adam(s):
    group, k = s["group"], s["step"] + 1
    b1, b2 = group["betas"]
    names = ("param", "master", "exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
    out = {n: s[n].double() for n in names if s[n] is not None}
    table = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()  # 0 ... 448, rising
    for t, (o, b, n) in enumerate(s["places"]):
        owner = torch.arange(n, device="cuda") // BLOCK
        part, blocks = slice(o, o + n), slice(b, b + int(owner[-1]) + 1)
        g = s["grad"][part].double()
        p = (s["param"] if s["master"] is None else s["master"])[part].double()
        m = b1 * s["exp_avg"][part].double() * s["exp_avg_scale"][blocks].double()[owner] + (1 - b1) * g
        v = b2 * (s["exp_avg_sq"][part].double() * s["exp_avg_sq_scale"][blocks].double()[owner]).square() + (1 - b2) * g.square()
        p = p * (1 - group["lr"] * group["weight_decay"]) - group["lr"] * (m / (1 - b1 ** k)) / ((v / (1 - b2 ** k)).sqrt() + group["eps"])
        out["param"][part] = p.to(s["param"].dtype).double()
        if s["master"] is not None:
            out["master"][part] = p
        bits = _bits(s["seed"], k, t, n)
        for name, x, u, power in (("exp_avg", m, bits & 0xFFFF, 1), ("exp_avg_sq", v.sqrt(), bits >> 16, 2)):
            most = torch.zeros(int(owner[-1]) + 1, dtype=torch.float64, device="cuda").scatter_reduce_(0, owner, x.abs(), "amax")
            scale = (most / 448).clamp(min=2.0 ** -126)
            y = (x.abs() / scale[owner]).clamp(max=448.0)
            above = torch.searchsorted(table, y, right=True).clamp(max=126)
            low, high = table[above - 1] ** power, table[above] ** power
            q = torch.where((u.double() + 0.5) / 65536 < (y ** power - low) / (high - low), table[above], table[above - 1])
            if power == 2:
                q = torch.where((x > 0) & (q == 0), table[1], q)
            out[name][part], out[name + "_scale"][blocks] = torch.sign(x) * q, scale
    return [out[n] for n in names if n in out]
