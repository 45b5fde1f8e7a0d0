from .softmax_xentropy import SoftmaxCrossEntropyLoss
from .token_loss import policy_loss, preference_loss, sequence_log_probs, token_log_probs

__all__ = [
    "SoftmaxCrossEntropyLoss",
    "policy_loss",
    "preference_loss",
    "sequence_log_probs",
    "token_log_probs",
]
