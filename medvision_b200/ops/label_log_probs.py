"""What a classifier answers at given labels: log-probability, entropy and the best alternatives, with their gradient."""
from typing import NamedTuple, Optional

import torch

from .. import _C


class LabelLogProbs(NamedTuple):
    log_prob: torch.Tensor
    entropy: torch.Tensor
    top_log_prob: Optional[torch.Tensor]
    top_label: Optional[torch.Tensor]


def label_log_probs(logits, labels, top=0):
    """Log-probabilities of ``labels`` under softmax(logits) over dimension 1, in one pass over the scores.

    Args:
        logits (Tensor): (N, classes) or (N, classes, [D,] H, W), float32, float16 or bfloat16
        labels (Tensor): (N, ...) or, as label fields are, (N, 1, ...), uint8, int16, int32 or int64; a value that is not a
            class (such as -1) stands for a label that is not given: log-probability 0, and no gradient from it
        top (int): number of alternatives, at most 16 and the number of classes

    Returns ``(log_prob, entropy, top_log_prob, top_label)``: float32 tensors of the labels' shape; the ``top`` largest
    log-probabilities and their classes (int32), (N, top, ...), ties to the lowest class, or None.  Differentiable in logits
    through log_prob and entropy; the alternatives carry no gradient.

    Scores of -inf are classes of probability 0.  Where all scores are -inf, log_prob is -inf, entropy 0 and the gradient 0.
    """
    return LabelLogProbs(*_C._native.label_log_probs(logits, labels, top))
