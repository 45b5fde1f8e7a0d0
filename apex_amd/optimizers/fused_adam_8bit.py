"""FusedAdam8bit — multi-tensor fused Adam/AdamW with both moments in 8 bits.

:class:`FusedAdam` holds 8 bytes of moments for every weight; this holds 2, with one fp32 scale for each 128
elements. For a model that is trained next to a frozen copy of itself (a reference to hold it near) that is the
memory of the copy.

A moment is ``scale * code`` with codes in ``torch.float8_e4m3fn``; the second moment is held as its root. Values
between two codes are rounded to one of them at random, with odds that keep the mean of the first and of the second
moment: rounded to nearest, a second moment with ``beta2 = 0.999`` would never move. The random numbers are a hash of
``(seed, step, tensor, element)``, so a run repeats bit for bit. The step itself is computed in fp32 from the new
moments before they are rounded. Device path: csrc/multi_tensor_adam_8bit.hip. CPU path: the same in plain torch.
"""

import math

import torch

from .._ext import get_ext
from ..tracing import traced
from ._scaling import found_inf_and_inv_scale

BLOCK = 128  # elements of one scale
_E4M3_MAX = 448.0
_MASK = 0xFFFFFFFF
_STATE = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")


def _mix(x):
    """32 mixed bits of an int, or of an int64 tensor (the kernel's mix32)."""
    x = x ^ (x >> 16)
    x = (x * 0x9E3779B1) & _MASK
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & _MASK
    return x ^ (x >> 16)


def _random_bits(seed, step, tensor, n):
    key = _mix((seed & _MASK) ^ _mix((step + _mix((tensor + 0x6A09E667) & _MASK)) & _MASK))
    i = torch.arange(n)
    return _mix((i * 0x9E3779B1 + key + (i >> 32) * 0x6A09E667) & _MASK)


def _in_blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _decode(codes, scales):
    n = codes.numel()
    return (_in_blocks(codes.float()) * scales[:, None]).view(-1)[:n]


def _encode(x, u, root):
    """Codes and scales of the fp32 values x; u in (0, 1) chooses between neighbours."""
    n = x.numel()
    finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
    scales = (_in_blocks(finite).amax(1) / _E4M3_MAX).clamp(min=torch.finfo(torch.float32).tiny)
    y = (_in_blocks(x) * (1.0 / scales)[:, None]).view(-1)[:n]
    size = y.abs().clamp(max=_E4M3_MAX)
    # the distance of codes at this size: 2^(exponent - 3), not under 2^-9
    step = torch.ldexp(torch.ones(()), torch.frexp(size.clamp(min=2.0 ** -6)).exponent - 4)
    z = size / step
    k = torch.floor(z)
    up = u * (2 * k + 1) < (z - k) * (z + k) if root else u < z - k
    k = k + up
    if root:
        k = torch.where((y > 0) & (k < 1), 1.0, k)
    q = torch.where(torch.isfinite(x), torch.copysign(k * step, y) + 0.0, math.nan)  # no code of -0
    return q.to(torch.float8_e4m3fn), scales


def _check_not_captured(device):
    """Before state is made: captured, it would be made anew at every replay."""
    if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("FusedAdam8bit makes its state, and after loading its masters, in a first step: take one before capture")


def _check_loaded(state, p):
    """Codes are met in memory order with a scale for each block: they have to lie as the param does."""
    if not all(k in state for k in _STATE):
        raise ValueError(f"FusedAdam8bit needs the state {_STATE} for each param, got {tuple(state)}")
    for name in _STATE + ("master_param",) * ("master_param" in state):
        v = state[name]
        scales = name.endswith("_scale")
        if v.dtype != (torch.float8_e4m3fn if name in ("exp_avg", "exp_avg_sq") else torch.float32):
            raise ValueError(f"FusedAdam8bit: {name} of a checkpoint is {v.dtype}")
        if v.shape != ((-(-p.numel() // BLOCK),) if scales else p.shape):
            raise ValueError(f"FusedAdam8bit: {name} of a checkpoint has shape {tuple(v.shape)} where the param's shape and "
                             f"layout are {tuple(p.shape)} and {p.stride()}")
        if not scales and any(n > 1 and a != b for n, a, b in zip(p.shape, v.stride(), p.stride())):
            raise ValueError(f"FusedAdam8bit: {name} of a checkpoint has another layout than the param: strides {v.stride()}, "
                             f"not {p.stride()}")


def _like(v, p):
    """A copy of state on the param's device; what has its shape gets its strides."""
    if v.shape != p.shape:
        return v.to(device=p.device).clone(memory_format=torch.preserve_format)
    return torch.empty_like(p, dtype=v.dtype, requires_grad=False).copy_(v)


class FusedAdam8bit(torch.optim.Optimizer):
    """Adam/AdamW with 8-bit moments in a single fused multi-tensor HIP kernel.

    Arguments are those of :class:`FusedAdam`, and

    - lr: with ``capturable`` a number becomes a tensor of each param group, to be changed in place; a tensor is used as
      it is, by all groups that set no other.
    - master_weights (bool): keep fp32 copies of fp16/bf16 params and step those (with or without ``capturable``).
      A step far smaller than a param's own spacing is lost without them.
    - seed (int): of the random rounding, kept in the param groups and so in checkpoints. Ranks that hold the same params
      need the same seed.

    Per param, ``state`` holds ``exp_avg`` and ``exp_avg_sq`` (``float8_e4m3fn`` codes of the param's shape;
    ``exp_avg_sq`` the root of the second moment), ``exp_avg_scale`` and ``exp_avg_sq_scale`` (fp32, one for each 128
    elements in memory order) and with ``master_weights`` ``master_param``. ``state_dict`` keeps them as they are. After a
    checkpoint without masters, ``master_weights`` makes them from the params in the first step; without it, a
    checkpoint's are left out.

    State is made in a param's first step, which cannot be captured; without ``capturable`` none can. Unlike
    :class:`FusedAdam` with ``capturable``, gradients are left as they are (not overwritten unscaled), and a
    step that GradScaler skips does not count.
    """

    def __init__(
        self,
        params,
        lr=1e-3,
        bias_correction=True,
        betas=(0.9, 0.999),
        eps=1e-8,
        adam_w_mode=True,
        weight_decay=0.0,
        amsgrad=False,
        set_grad_none=True,
        capturable=False,
        master_weights=False,
        seed=0,
    ):
        if amsgrad:
            raise RuntimeError("FusedAdam8bit does not support the AMSGrad variant.")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must be in [0, 1), got {betas}")
        if not eps >= 0.0:
            raise ValueError(f"eps must not be negative, got {eps}")
        self.capturable = capturable  # groups are added by it
        defaults = dict(lr=lr, bias_correction=bias_correction, betas=betas, eps=eps, weight_decay=weight_decay,
                        seed=int(seed))
        super().__init__(params, defaults)
        self.adam_w_mode = 1 if adam_w_mode else 0
        self.set_grad_none = set_grad_none
        self.master_weights = master_weights
        self._step_supports_amp_scaling = capturable

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        if self.capturable and not torch.is_tensor(group["lr"]):
            # the kernel reads it on the device, so that a hipGraph's replay sees new values; schedules write it in
            # place, so each group has its own
            params = group["params"]
            device = params[0].device if params else "cuda" if torch.cuda.is_available() else "cpu"
            group["lr"] = torch.tensor(group["lr"], dtype=torch.float32, device=device)

    def zero_grad(self, set_to_none: bool = True):
        super().zero_grad(set_to_none=self.set_grad_none or set_to_none)

    def load_state_dict(self, state_dict):
        # torch casts state to the params' type: the codes and scales are put back as they were saved
        saved = state_dict["state"]
        order = [k for g in state_dict["param_groups"] for k in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for k, p in zip(order, params):
            if saved.get(k):
                _check_loaded(saved[k], p)
        super().load_state_dict(state_dict)
        for k, p in zip(order, params):
            if k in saved:
                self.state[p] = {
                    name: _like(v, p) if torch.is_tensor(v) else v
                    for name, v in saved[k].items()
                    if name != "master_param" or self.master_weights
                }
        for group in self.param_groups:
            group.setdefault("seed", self.defaults["seed"])  # of a checkpoint that does not keep it
        if self.capturable:
            for group in self.param_groups:
                if group["params"]:
                    device = group["params"][0].device
                    for key, dtype in (("lr", torch.float32), ("step", torch.int32)):
                        v = group.get(key)
                        if v is not None:
                            group[key] = torch.as_tensor(v, dtype=dtype, device=device).clone()  # groups may share it
        else:
            for group in self.param_groups:
                for key in ("lr", "step"):
                    if torch.is_tensor(group.get(key)):
                        group[key] = group[key].item()

    def _init_state(self, p, state):
        if p.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            raise RuntimeError("FusedAdam8bit only supports fp16/bf16/fp32 params")
        if torch.empty_like(p, device="meta").stride() != p.stride():
            raise RuntimeError("FusedAdam8bit only supports dense params without gaps or overlaps")
        _check_not_captured(p.device)
        blocks = -(-p.numel() // BLOCK)
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
            state[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)

    def _init_master(self, p, state):
        _check_not_captured(p.device)
        state["master_param"] = p.detach().float().clone()

    @torch.no_grad()
    @traced("FusedAdam8bit.step")
    def step(self, closure=None, grad_scaler=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()

        founds = unscale = None
        if self.capturable and grad_scaler is not None:
            founds, unscale = found_inf_and_inv_scale(self, grad_scaler)
        masters = self.master_weights
        first = 0  # a tensor's place in the optimizer is part of its random numbers
        for group in self.param_groups:
            params = group["params"]
            if not params:
                continue
            lists = {}  # by device, dtype and whether there is a master copy
            for place, p in enumerate(params, first):
                grad = p.grad
                if grad is None:
                    continue
                if grad.is_sparse:
                    raise RuntimeError("FusedAdam8bit does not support sparse gradients")
                state = self.state[p]
                if not state:
                    self._init_state(p, state)
                if masters and "master_param" not in state and p.dtype != torch.float32:
                    self._init_master(p, state)  # new, or loaded from a checkpoint without
                key = p.device, p.dtype, "master_param" in state
                row = place, grad, p, state
                if key in lists:
                    lists[key].append(row)
                else:
                    lists[key] = [row]
            first += len(params)
            found_inf, inv_scale = self._count(group, founds, unscale)
            for (device, _, master), rows in lists.items():
                names = _STATE + (("master_param",) if master else ())
                if device.type == "cuda":
                    tensors = [[r[1] for r in rows], [r[2] for r in rows]] + [[r[3][name] for r in rows] for name in names]
                    self._step_cuda(group, [r[0] for r in rows], tensors, found_inf, inv_scale)
                elif found_inf is None or not float(found_inf):
                    for place, grad, p, state in rows:
                        if grad.stride() != p.stride():  # elements are met in memory order
                            grad = torch.empty_like(p).copy_(grad)
                        self._step_ref(group, place, inv_scale, grad, p, *(state[name] for name in names))
        return loss

    def _count(self, group, founds, inv_scale):
        """Advances the group's step; what GradScaler has for it, on its device."""
        device = group["params"][0].device
        if not self.capturable:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("FusedAdam8bit needs capturable=True to be captured: replays would repeat one step's numbers")
            group["step"] = group.get("step", 0) + 1
            return None, None
        if "step" not in group:
            _check_not_captured(device)
            group["step"] = torch.zeros(1, dtype=torch.int32, device=device)
        if torch.is_tensor(group["lr"]) and group["lr"].device != device:
            group["lr"] = group["lr"].to(device)
        if not founds:
            group["step"].add_(1)  # in place: a hipGraph's replay has to see it
            return None, None
        # a gradient on any device that is not finite skips the step on all
        found = [f.to(device=device, dtype=torch.float32) for f in founds.values()]
        found_inf = found[0] if len(found) == 1 else torch.stack(found).amax(0)
        group["step"].add_((found_inf == 0).to(torch.int32))
        return found_inf, inv_scale if inv_scale is None else inv_scale.to(device)

    # ----- device path -----
    def _step_cuda(self, group, places, tensors, found_inf, inv_scale):
        amp_C = get_ext("amp_C")
        beta1, beta2 = group["betas"]
        bias_correction = 1 if group["bias_correction"] else 0
        if self.capturable:
            lr = group["lr"]
            if not torch.is_tensor(lr):  # a schedule wrote a number
                lr = group["lr"] = torch.tensor(lr, dtype=torch.float32, device=tensors[0][0].device)
            amp_C.multi_tensor_adam_8bit_capturable(
                tensors, places, lr.float(), beta1, beta2, group["eps"], group["step"], self.adam_w_mode,
                bias_correction, group["weight_decay"], group["seed"] & _MASK, inv_scale, found_inf)
        else:
            amp_C.multi_tensor_adam_8bit(
                tensors, places, float(group["lr"]), beta1, beta2, group["eps"], group["step"], self.adam_w_mode,
                bias_correction, group["weight_decay"], group["seed"] & _MASK)

    # ----- reference path (CPU CI + numerics oracle) -----
    def _step_ref(self, group, place, inv_scale, g, p, m, m_scale, r, r_scale, master=None):
        step, lr = int(group["step"]), float(group["lr"])
        beta1, beta2 = group["betas"]
        bc1 = 1.0 - beta1 ** step if group["bias_correction"] else 1.0
        bc2 = 1.0 - beta2 ** step if group["bias_correction"] else 1.0
        wd = group["weight_decay"]

        def flat(t):  # memory order
            return t.as_strided((t.numel(),), (1,))

        n = p.numel()
        if n == 0:
            return
        bits = _random_bits(group["seed"], step, place, n)
        gf = flat(g).float() * (1.0 if inv_scale is None else float(inv_scale))
        pf = flat(p if master is None else master).float()
        if self.adam_w_mode == 0:
            gf = gf + wd * pf
        mf = beta1 * _decode(flat(m), m_scale) + (1 - beta1) * gf
        rf = _decode(flat(r), r_scale)
        rf = (beta2 * rf * rf + (1 - beta2) * gf * gf).sqrt()  # in the kernel's order
        update = (mf / bc1) / (rf / math.sqrt(bc2) + group["eps"])
        if self.adam_w_mode == 1:
            update = update + wd * pf
        pf = pf - lr * update
        flat(p).copy_(pf)
        if master is not None:
            flat(master).copy_(pf)
        for x, u, codes, scales, root in ((mf, bits & 0xFFFF, m, m_scale, False), (rf, bits >> 16, r, r_scale, True)):
            q, s = _encode(x, (u.float() + 0.5) / 65536, root)
            flat(codes).copy_(q)
            scales.copy_(s)
