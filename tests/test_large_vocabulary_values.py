"""Cross entropy against a vocabulary (ops.linear_cross_entropy) with elements and factors far from ordinary: infinite classes, rows whose losses count very differently.  Plain form and
tolerances are those of the operator's other tests."""
import pytest
import torch

from lookahead_keys_attention_amd import ops
from test_vocab import DEV, TYPES, gpu, inputs, reference, within


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [8, 24, 72, 96, 128, 520])
def test_a_class_of_minus_infinity_has_no_weight(D, dtype):
    """One element of a class is -inf and meets positive elements in every row: its logits are -inf, whatever the width; loss and the table's gradient are those without the class."""
    R, V, gone = 70, 300, 37
    x, w, target = inputs(R, V, D, dtype, D)
    target[target == gone] = gone + 1
    x[:, D - 3] = x[:, D - 3].abs() + 0.5
    rest = [v for v in range(V) if v != gone]
    masked = w.clone()
    masked[gone, D - 3] = -float("inf")
    one = torch.ones((), dtype=dtype, device=DEV)
    ref = reference(x, w[rest], torch.where(target > gone, target - 1, target), "mean", one, -100, dtype)
    leaf = masked.requires_grad_()
    loss = ops.linear_cross_entropy(x, leaf, target)
    dw, = torch.autograd.grad(loss, leaf, one)
    within(loss.detach(), *ref[0], dtype, "loss")
    within(dw[rest], *ref[2], dtype, "dw")
    assert not dw[gone].any()
