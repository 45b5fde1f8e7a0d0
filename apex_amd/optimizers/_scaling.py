"""What an optimizer that takes ``torch.amp.GradScaler`` itself (``_step_supports_amp_scaling``) asks it in a step."""

from torch.amp.grad_scaler import OptState


def found_inf_and_inv_scale(optimizer, grad_scaler):
    """Which devices' gradients are not finite, and ``1 / scale``: ``None`` where ``grad_scaler.unscale_`` has divided
    the gradients already. Reads and writes all gradients of the optimizer, unless ``unscale_`` has looked at them."""
    state = grad_scaler._per_optimizer_states[id(optimizer)]
    if state["stage"] is OptState.UNSCALED:
        return state["found_inf_per_device"], None
    found_inf = grad_scaler._check_inf_per_device(optimizer)
    return found_inf, grad_scaler._get_scale_async().double().reciprocal().float()
