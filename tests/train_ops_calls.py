"""Calls of the training operators that differ in one argument."""
import torch

from litnicelm_b200 import training


def calls_with(x, other):
    """Every operator with x in each place in turn that takes a tensor of its shape ([1, 4, 2, 8] or [2, 8]), and `other` in the rest."""
    y, dev = other, x.device
    if x.dim() == 4:
        lse = torch.zeros(1, 2, 4, device=dev)
        return [lambda: training.attention_forward(x, y, y), lambda: training.attention_forward(y, x, y),
                lambda: training.attention_forward(y, y, x), lambda: training.attention_forward(y, y, y, out=x),
                lambda: training.attention_backward(x, y, y, y, y, lse), lambda: training.attention_backward(y, x, y, y, y, lse),
                lambda: training.attention_backward(y, y, y, y, x, lse), lambda: training.attention_backward(y, y, y, y, y, lse, dq=x),
                lambda: training.attention_backward(y, y, y, y, y, lse, dk=x),
                lambda: training.attention_backward(y, y, y, y, y, lse, dv=x)]
    ids, n = torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(2, device=dev)
    return [lambda: training.policy_loss(x, ids, n, n), lambda: training.policy_loss(y, ids, n, n, dlogits=x),
            lambda: training.orthogonalise(x), lambda: training.orthogonalise(y, out=x), lambda: training.muon_step(x, y, y, 0.1),
            lambda: training.muon_step(y, x, y, 0.1), lambda: training.muon_step(y, y, x, 0.1)]
