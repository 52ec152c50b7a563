"""Cross entropy against a vocabulary (ops.linear_cross_entropy) with elements and factors far from ordinary: infinite classes, rows whose losses count very differently.  Plain form and
tolerances are those of the operator's other tests."""
import pytest
import torch

from lookahead_keys_attention_amd import ops
from test_vocab import DEV, TYPES, U, gpu, inputs, reference, within


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


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_whose_losses_count_very_differently(dtype):
    """Each row's gradient is as exact as the row's own factor allows, however small that is beside the others', an infinite one among them; a table of one sign, so that what many unlikely
    classes add is a large part of it.  d of a row lies in the type under a factor of 2^10 at least (fp16), so what is below its normal numbers is off by 2^-25 / 2^10 of the row's own
    factor; the table's gradient has that of the largest, twice: d is rounded again where it goes to the common factor."""
    R, V, D = 150, 9000, 64
    g = torch.Generator().manual_seed(21)
    x, w, target = inputs(R, V, D, dtype, 21)
    w = (w.float().abs() + 0.25).to(dtype)
    x = (x.float() / 16).to(dtype)
    low, high = (-9, 14) if dtype is torch.float16 else (-60, 30)
    dloss = (2.0 ** torch.randint(low, high + 1, (R,), generator=g).double() * (1 + torch.rand(R, generator=g).double())).to(dtype).to(DEV)
    dloss[:2] = torch.tensor([2.0 ** low, 2.0 ** high])
    target[5] = -100
    keep = target != -100
    leaves = [x.requires_grad_(), w.requires_grad_()]
    each = ops.linear_cross_entropy(*leaves, target, "none")
    dx, dw = torch.autograd.grad(each, leaves, dloss, retain_graph=True)
    for r in range(R):   # a row by itself: its factor is the largest
        if keep[r]:
            (_, _), (ref, bound), _ = reference(x[r:r + 1].detach(), w.detach(), target[r:r + 1], "none", dloss[r:r + 1], -100, dtype)
            if dtype is torch.float16:
                bound = bound + 2.0 ** -35 * dloss[r].double().abs() * w.detach().double().abs().sum(0)
            within(dx[r:r + 1], ref, bound, dtype, (r, dloss[r].item()))
    assert not dx[5].any()
    (_, _), _, (ref, bound) = reference(x.detach(), w.detach(), target, "none", dloss, -100, dtype)
    if dtype is torch.float16:
        bound = bound + 2.0 ** -25 / 2.0 ** 14 * dloss[keep].double().abs().max() * x.detach()[keep].double().abs().sum(0)
    within(dw, ref, bound, dtype, "dw")
    # alone of all, one gradient without the other: the same bits
    assert torch.equal(torch.autograd.grad(each, leaves[1], dloss, retain_graph=True)[0], dw)
    assert torch.equal(torch.autograd.grad(each, leaves[0], dloss, retain_graph=True)[0], dx)
    # an infinite factor is its row's alone, as far as the rows' gradients go
    dloss[3] = float("inf")
    again, = torch.autograd.grad(each, leaves[0], dloss)
    others = torch.arange(R, device=DEV) != 3
    assert not again[3].isfinite().any()
    for r in (0, 1, 40, 149):
        (_, _), (ref, bound), _ = reference(x[r:r + 1].detach(), w.detach(), target[r:r + 1], "none", dloss[r:r + 1], -100, dtype)
        if dtype is torch.float16:
            bound = bound + 2.0 ** -35 * dloss[r].double().abs() * w.detach().double().abs().sum(0)
        within(again[r:r + 1], ref, bound, dtype, (r, "beside an infinite one"))
    assert again[others].isfinite().all()


@gpu
def test_rows_whose_losses_count_very_differently_in_several_pieces():
    """The same in fp16 over a vocabulary of two pieces of d."""
    R, V, D, dtype = 4200, 140001, 16, torch.float16
    g = torch.Generator().manual_seed(22)
    x, w, target = inputs(R, V, D, dtype, 22)
    w = (w.float().abs() + 0.25).to(dtype)
    dloss = (2.0 ** torch.randint(-9, 15, (R,), generator=g).double()).to(dtype).to(DEV)
    dloss[::3] = 0
    target[::7] = -100
    leaves = [x.requires_grad_(), w.requires_grad_()]
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(*leaves, target, "none"), leaves, dloss)
    x, w = x.detach(), w.detach()
    for r in [int(dloss[r] != 0) and r for r in (1, 2, 4, 64, 100, 2000, 4199)]:
        _, (ref, bound), _ = reference(x[r:r + 1], w, target[r:r + 1], "none", dloss[r:r + 1], -100, dtype)
        within(dx[r:r + 1], ref, bound + 2.0 ** -35 * dloss[r].double().abs() * w.double().abs().sum(0), dtype, (r, dloss[r].item()))
    assert not dx[::3].any() and not dx[::7].any()
    _, _, (ref, bound) = reference(x, w, target, "none", dloss, -100, dtype)
    within(dw, ref, bound + 2.0 ** -25 / 2.0 ** 14 * dloss.double().abs().max() * x[target != -100].double().abs().sum(0), dtype, "dw")


@gpu
def test_the_backward_operator_refuses_what_no_forward_pass_has_returned():
    x, w, target = inputs(20, 30, 16, torch.bfloat16, 23)
    forward, backward = torch.ops.castle_hip.linear_cross_entropy, torch.ops.castle_hip.linear_cross_entropy_bwd
    loss, state = forward(x, w, target, 0, -100)
    good = backward(loss, x, w, target, state, 0, -100)
    for bad in (state.cpu(), state.view(torch.int32), state[None], state.repeat_interleave(2)[::2]):
        with pytest.raises(ValueError, match="state"):
            backward(loss, x, w, target, bad, 0, -100)
    for bad in (state[:-256], torch.cat((state[:16], state))[16:], state[:0]):   # too short, not at 256 bytes
        with pytest.raises(RuntimeError):
            backward(loss, x, w, target, bad, 0, -100)
    assert all(torch.equal(a, b) for a, b in zip(backward(loss, x, w, target, state.clone(), 0, -100), good))


@gpu
@pytest.mark.parametrize("R", [1, 2, 7, 33, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_rows_lose_nothing_of_their_targets(R, dtype, reduction):
    """Each row has eight columns of its own, in it and in the class it aims at, and other classes are zero: in these columns both gradients are the target's part alone, which is p - 1 of
    32 bits times the factor, the logit off by ez as everywhere, and is rounded once.  Some rows have the same target, one does not count, one's is not there."""
    D, V = 8 * max(R, 3), 5000
    g = torch.Generator().manual_seed(R)
    target = torch.randint(0, V, (R,), generator=g)
    target[3::5] = target[0]
    own = torch.arange(D)[None] // 8 == torch.arange(R)[:, None]
    x = torch.where(own, torch.randn(R, D, generator=g), 0.0).to(dtype)
    w = torch.zeros(V, D)
    for r in range(R):   # (logits of 4 to 12: softmax values of the target from 0.01 to 0.97)
        v = torch.randn(8, generator=g)
        part = x[r, own[r]].float()
        w[target[r], own[r]] = v + (4 + 8 * torch.rand(1, generator=g) - v @ part) * part / (part @ part)
    w = w.to(dtype)
    counts = torch.ones(R, dtype=torch.bool)
    if R > 8:
        counts[5] = False
    given = torch.where(counts, target, -100)
    dloss = torch.tensor(0.8125, dtype=dtype) if reduction == "mean" else (0.5 + torch.rand(R, generator=g)).to(dtype)
    if reduction == "none" and dtype is torch.float16:
        dloss[R // 2] *= 2.0 ** -9   # (a power of two of its own)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w)]
    loss = ops.linear_cross_entropy(*leaves, given.to(DEV), reduction)
    dx, dw = (t.cpu().double() for t in torch.autograd.grad(loss, leaves, dloss.to(DEV), retain_graph=True))
    assert torch.equal(torch.autograd.grad(loss, leaves[0], dloss.to(DEV), retain_graph=True)[0].cpu().double(), dx)
    assert torch.equal(torch.autograd.grad(loss, leaves[1], dloss.to(DEV))[0].cpu().double(), dw)
    x, w = x.double(), w.double()
    z, half = x @ w.T, torch.finfo(dtype).eps / 2
    lse = torch.logsumexp(z, 1)
    for r in range(R):
        if not counts[r]:
            assert not dx[r].any()
            continue
        factor, p = dloss.double().expand(R)[r] / (counts.sum() if reduction == "mean" else 1), torch.exp(z[r, target[r]] - lse[r])
        ez = (D / 16 + 32) * U * (x[r].abs() @ w[target[r]].abs())
        off = abs(factor) * (p * (2 * ez + 16 * U * (1 + lse[r].abs())) + 8 * U)
        for got, other in ((dx[r, own[r]], w[target[r], own[r]]), (dw[target[r], own[r]], x[r, own[r]])):
            ref = factor * (p - 1) * other
            most = off * other.abs() + half * (ref.abs() + off * other.abs()).clamp(min=torch.finfo(dtype).tiny)
            assert ((got - ref).abs() <= most).all(), (r, ((got - ref).abs() / most).max())
