"""Losses on the log-probabilities of given tokens: what a language model is scored and trained with after its
first training.

- :func:`token_log_probs`, :func:`sequence_log_probs`: how likely the model finds given tokens, or whole answers.
- :func:`preference_loss`: paired log ratios of a chosen and a rejected answer against a frozen reference.
- :func:`policy_loss`: the clipped ratio loss with a KL term.

All take logits ``[..., V]`` (fp32, fp16 or bf16) and labels of the leading shape: ``labels[i]`` is the token whose
log-probability row ``i`` of the logits gives, so a causal model's labels are its tokens moved one place to the left.
Rows whose label is ``ignore_index`` (prompts, padding) are not read and get no gradient, whatever they hold; rows
whose gradient turns out to be 0 (clipped tokens) are not read in the backward pass.

On the GPU a loss is one pass over the logits, which keeps two floats of each row, a small pass over the rows'
log-probabilities, and in the backward pass one more read of the logits while their gradient is written: no
``[..., V]`` intermediate is ever stored (csrc/token_loss.hip). Sums over tokens are kept in 64 bits, all reductions
in a fixed order. A label outside ``[0, V)`` gives NaN there (the host does not wait to look at it); on the CPU it
raises. Passes can be captured into a hipGraph.
"""

import math

import torch

from ..._ext import get_ext

_KINDS = {"sigmoid": 0, "ipo": 1, "hinge": 2}
_REDUCTIONS = {"token": 0, "sequence": 1, "sum": 2, "none": 3}


# ---- checks ----


def _check(logits, labels, ignore_index, temperature=1.0):
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise TypeError(f"logits must be fp32, fp16 or bf16, got {logits.dtype}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"labels must be int64 or int32, got {labels.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits need a last dimension of the vocabulary, got {tuple(logits.shape)}")
    if labels.shape != logits.shape[:-1]:
        raise ValueError(f"labels must have shape {tuple(logits.shape[:-1])}, got {tuple(labels.shape)}")
    if labels.device != logits.device:
        raise ValueError(f"labels are on {labels.device}, logits on {logits.device}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be in [1e-6, 1e6], got {temperature}")
    return labels.contiguous() if labels.dtype == torch.int64 else labels.long().contiguous()


def _check_sequences(labels, cu_seqlens):
    """The number of sequences: rows of 2-D labels, or what cu_seqlens says of 1-D ones."""
    if cu_seqlens is None:
        if labels.dim() != 2:
            raise ValueError(f"labels must be [sequences, length], or 1-D with cu_seqlens, got {tuple(labels.shape)}")
        return labels.shape[0]
    if labels.dim() != 1:
        raise ValueError(f"with cu_seqlens labels must be 1-D, got {tuple(labels.shape)}")
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype != torch.int32:
        raise ValueError("cu_seqlens must be 1-D int32 with one value more than there are sequences")
    if not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be contiguous")
    if cu_seqlens.device != labels.device:
        raise ValueError(f"cu_seqlens are on {cu_seqlens.device}, labels on {labels.device}")
    return cu_seqlens.numel() - 1


def _given(t, name, like, *shapes):
    """`t` in fp32 and contiguous; it has to have one of the shapes."""
    if t.shape not in shapes:
        raise ValueError(f"{name} must have shape {' or '.join(str(tuple(s)) for s in shapes)}, got {tuple(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point, got {t.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, logits on {like.device}")
    return t.detach() if t.dtype == torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


# ---- CPU path: plain torch, differentiated by autograd ----


def _ref_log_probs(logits, labels, ignore_index, temperature):
    on = labels != ignore_index
    rows = torch.log_softmax(logits[on].float() / temperature, dim=-1)
    picked = rows.gather(-1, labels[on].unsqueeze(-1)).squeeze(-1)
    return torch.zeros(labels.shape, dtype=torch.float32).masked_scatter(on, picked)


def _ref_owner(labels, cu_seqlens):
    """Each token's sequence, and which tokens have one."""
    at = torch.arange(labels.numel())
    if cu_seqlens is None:
        return at // max(1, labels.shape[1]), torch.ones_like(at, dtype=torch.bool)
    cu = cu_seqlens.long().clamp(0, labels.numel())
    owner = torch.bucketize(at, cu[1:], right=True)
    inside = (at >= cu[0]) & (owner < cu.numel() - 1)
    return owner.clamp(max=cu.numel() - 2), inside


def _ref_sums(lp, labels, ignore_index, cu_seqlens, count, average):
    owner, inside = _ref_owner(labels, cu_seqlens)
    on = inside & (labels != ignore_index).view(-1)
    sums = torch.zeros(count, dtype=torch.float64).index_add(0, owner[on], lp.reshape(-1)[on].double())
    if average:
        sums = sums / torch.bincount(owner[on], minlength=count).clamp(min=1)
    return sums


# ---- log-probabilities ----


def token_log_probs(logits, labels, ignore_index=-100, temperature=1.0):
    """Log-probability of each label under ``softmax(logits / temperature)``: fp32, of the labels' shape, 0 where the
    label is ``ignore_index``. Differentiable in the logits."""
    labels = _check(logits, labels, ignore_index, temperature)
    if logits.is_cuda:
        return get_ext("token_loss").token_log_probs(logits, labels, ignore_index, temperature)
    return _ref_log_probs(logits, labels, ignore_index, temperature)


def sequence_log_probs(logits, labels, cu_seqlens=None, average=False, ignore_index=-100, temperature=1.0):
    """Log-probability of each sequence, the sum (or with ``average`` the mean) over its labelled tokens: fp32
    ``[sequences]``, 0 for a sequence without one. Sequences are the rows of 2-D labels, or with 1-D labels rows
    ``cu_seqlens[s]`` to ``cu_seqlens[s + 1]`` (int32). Differentiable in the logits. Under ``torch.no_grad()`` on the
    reference's logits it gives :func:`preference_loss` its ``ref_log_probs``."""
    labels = _check(logits, labels, ignore_index, temperature)
    count = _check_sequences(labels, cu_seqlens)
    if logits.is_cuda:
        return get_ext("token_loss").sequence_log_probs(logits, labels, cu_seqlens, count, bool(average), ignore_index, temperature)
    lp = _ref_log_probs(logits, labels, ignore_index, temperature)
    return _ref_sums(lp, labels, ignore_index, cu_seqlens, count, average).float()


# ---- paired log ratios ----


def preference_loss(logits, labels, ref_log_probs, beta=0.1, label_smoothing=0.0, loss_type="sigmoid", average=False,
                    cu_seqlens=None, ignore_index=-100):
    """Preference loss over pairs of answers: the first half of the sequences was chosen, the second half rejected,
    pair ``b`` being sequences ``b`` and ``pairs + b``.

    With the sequences' log-probabilities under the policy and the reference (summed over labelled tokens, with
    ``average`` their mean) and ``d = (policy - ref)[chosen] - (policy - ref)[rejected]``, the loss is the pairs' mean of

    - ``"sigmoid"``: ``-(1 - label_smoothing) log sigmoid(beta d) - label_smoothing log sigmoid(-beta d)``
    - ``"ipo"``: ``(d - 1 / (2 beta)) ** 2``
    - ``"hinge"``: ``max(0, 1 - beta d)``

    Args:
        logits: ``[2 * pairs, length, V]``, or with ``cu_seqlens`` ``[tokens, V]``.
        ref_log_probs: ``[2 * pairs]``, as :func:`sequence_log_probs` gives them (with the same ``average``).
        cu_seqlens: int32 ``[2 * pairs + 1]``, the sequences' first tokens, which do not fall; tokens outside them have
            no part.

    Returns:
        ``(loss, chosen_rewards, rejected_rewards)``: the loss, differentiable in the logits, and
        ``beta * (policy - ref)`` of each answer, ``[pairs]``, which are not.
    """
    labels = _check(logits, labels, ignore_index)
    count = _check_sequences(labels, cu_seqlens)
    if count % 2 or count == 0 or labels.numel() == 0:
        raise ValueError(f"preference_loss needs pairs of sequences with tokens, got {count} sequences, {labels.numel()} tokens")
    if loss_type not in _KINDS:
        raise ValueError(f"loss_type must be one of {sorted(_KINDS)}, got {loss_type!r}")
    if not (math.isfinite(beta) and beta > 0):
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing < 0.5:
        raise ValueError(f"label_smoothing must be in [0, 0.5), got {label_smoothing}")
    if label_smoothing and loss_type != "sigmoid":
        raise ValueError("label_smoothing goes with loss_type='sigmoid' only")
    ref = _given(ref_log_probs, "ref_log_probs", logits, (count,))
    pairs = count // 2
    if logits.is_cuda:
        return tuple(get_ext("token_loss").preference_loss(logits, labels, ref, cu_seqlens, pairs, _KINDS[loss_type], beta,
                                                           label_smoothing, bool(average), ignore_index))
    lp = _ref_log_probs(logits, labels, ignore_index, 1.0)
    gain = _ref_sums(lp, labels, ignore_index, cu_seqlens, count, average) - ref.double()
    z = beta * (gain[:pairs] - gain[pairs:])
    if loss_type == "sigmoid":
        softplus = torch.nn.functional.softplus
        loss = (1 - label_smoothing) * softplus(-z, threshold=1e9)
        if label_smoothing:
            loss = loss + label_smoothing * softplus(z, threshold=1e9)
    elif loss_type == "ipo":
        loss = (z / beta - 0.5 / beta) ** 2
    else:
        loss = torch.where(z >= 1, 0.0, 1 - z)
    rewards = (beta * gain).detach().float()
    return loss.mean().float(), rewards[:pairs], rewards[pairs:]


# ---- clipped policy loss ----


def policy_loss(logits, labels, old_log_probs, advantages, ref_log_probs=None, clip_eps=0.2, clip_eps_high=None,
                kl_coef=0.0, temperature=1.0, reduction="token", cu_seqlens=None, ignore_index=-100, grad_scale=None):
    """Clipped policy loss with a KL term against a reference.

    For a labelled token with log-probability ``lp``, ``ratio = exp(lp - old)``, advantage ``A`` and ``d = ref - lp``::

        loss = -min(ratio A, clamp(ratio, 1 - clip_eps, 1 + clip_eps_high) A) + kl_coef (exp(d) - d - 1)

    Args:
        logits: ``[sequences, length, V]``, or ``[tokens, V]`` with 1-D labels.
        old_log_probs: of the policy that the tokens were drawn from, of the labels' shape (at the same
            ``temperature``); ``None`` if it is this one (``ratio`` is 1, its gradient is that of ``lp``).
        advantages: of the labels' shape, or ``[sequences]`` or ``[sequences, 1]``. Of as many packed sequences as tokens
            ``[sequences]`` is the labels' shape and goes by token: ``[sequences, 1]`` goes by sequence there too.
        ref_log_probs: of the labels' shape; needed where ``kl_coef`` is not 0.
        clip_eps_high: the upper clip, ``clip_eps`` if ``None``.
        reduction: ``"token"``, the mean over all labelled tokens; ``"sequence"``, the mean over all sequences of their
            tokens' mean (0 for a sequence without one); ``"sum"``; ``"none"``, the loss of each token.
        cu_seqlens: int32 ``[sequences + 1]``, for 1-D labels; tokens outside have no part. Without it, 1-D labels are
            one sequence.
        grad_scale: a number, or a tensor of one fp32 value on the logits' device, finite and not 0. Where it is given,
            the forward pass also makes the logits' gradient, for a loss that is going to be multiplied by
            ``grad_scale`` before ``backward()`` (1 if it is not), and where a row fits a compute unit's registers it
            reads the logits only once. It keeps that gradient in place of the logits. If another gradient of the loss
            arrives, the kept one is multiplied by their quotient. The backward pass can then be run once only.

    Returns:
        ``(loss, log_probs)``: the loss, differentiable in the logits, and the tokens' log-probabilities, fp32 of the
        labels' shape, which are not (0 where the label is ``ignore_index``).
    """
    labels = _check(logits, labels, ignore_index, temperature)
    if cu_seqlens is None and labels.dim() == 1:
        count = 1
    else:
        count = _check_sequences(labels, cu_seqlens)
    if count == 0 or labels.numel() == 0:
        raise ValueError(f"policy_loss needs a sequence with a token, got labels of {tuple(labels.shape)}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTIONS)}, got {reduction!r}")
    high = clip_eps if clip_eps_high is None else clip_eps_high
    if not (0 <= clip_eps <= 1 and 0 <= high < math.inf):
        raise ValueError(f"clip_eps must be in [0, 1] and clip_eps_high not negative, got {clip_eps} and {high}")
    if not (math.isfinite(kl_coef) and kl_coef >= 0):
        raise ValueError(f"kl_coef must not be negative, got {kl_coef}")
    if kl_coef and ref_log_probs is None:
        raise ValueError("kl_coef needs ref_log_probs")
    old = None if old_log_probs is None else _given(old_log_probs, "old_log_probs", logits, labels.shape)
    ref = None if ref_log_probs is None or not kl_coef else _given(ref_log_probs, "ref_log_probs", logits, labels.shape)
    by_row = advantages.shape == labels.shape
    advantages = _given(advantages, "advantages", logits, labels.shape, (count,), (count, 1))
    if grad_scale is not None:
        if reduction == "none":
            raise ValueError("grad_scale goes with a loss that is one number: not with reduction='none'")
        if torch.is_tensor(grad_scale):
            if grad_scale.numel() != 1 or grad_scale.dtype != torch.float32 or grad_scale.device != logits.device:
                raise ValueError("grad_scale must be a number, or one fp32 value on the logits' device")
        elif not (math.isfinite(grad_scale) and grad_scale != 0):
            raise ValueError(f"grad_scale must be finite and not 0, got {grad_scale}")
    args = (labels, old, advantages, by_row, ref, cu_seqlens, count, clip_eps, high, kl_coef, temperature,
            _REDUCTIONS[reduction], ignore_index)
    if logits.is_cuda:
        tensor = grad_scale.detach().reshape(1) if torch.is_tensor(grad_scale) else None
        number = 1.0 if tensor is not None or grad_scale is None else grad_scale
        return tuple(get_ext("token_loss").policy_loss(logits, *args, grad_scale is not None, number, tensor))
    lp = _ref_log_probs(logits, labels, ignore_index, temperature)
    return _ref_policy(lp, *args)


class _One(torch.autograd.Function):
    """exp(x - x) with x's gradient: 1, where x is -inf as well."""

    @staticmethod
    def forward(ctx, x):
        one = torch.where(torch.isnan(x), x, 1.0)
        ctx.save_for_backward(one)
        return one

    @staticmethod
    def backward(ctx, grad):
        return grad * ctx.saved_tensors[0]


def _ref_policy(lp, labels, old, advantages, by_row, ref, cu_seqlens, count, low, high, kl, temperature, reduction, ignore_index):
    if cu_seqlens is None and labels.dim() == 1:
        owner, inside = torch.zeros_like(labels), torch.ones_like(labels, dtype=torch.bool)
    else:
        owner, inside = _ref_owner(labels, cu_seqlens)
    on = inside & (labels != ignore_index).view(-1)
    x, owner = lp.reshape(-1)[on], owner[on]
    a = advantages.view(-1)[on if by_row else owner]
    ratio = _One.apply if old is None else lambda z: torch.exp(z - old.view(-1)[on])
    now = ratio(x.detach())
    bound = now.clamp(1 - low, 1 + high) * a
    held = now * a > bound
    # a token that the clip holds has no gradient: not that of a ratio of inf, times 0, either
    each = -torch.where(held, bound, ratio(torch.where(held, x.detach(), x)) * a)
    if ref is not None:
        d = ref.view(-1)[on] - x
        each = each + kl * (torch.expm1(d) - d)
    each, lp = each.double(), lp.detach()
    if reduction == _REDUCTIONS["none"]:
        return torch.zeros(labels.shape).masked_scatter(on.view(labels.shape), each.float()), lp
    if reduction == _REDUCTIONS["sequence"]:
        sums = torch.zeros(count, dtype=torch.float64).index_add(0, owner, each)
        loss = (sums / torch.bincount(owner, minlength=count).clamp(min=1)).mean()
    else:
        loss = each.sum() / (max(1, each.numel()) if reduction == _REDUCTIONS["token"] else 1)
    return loss.float(), lp
