"""Cross entropy against a vocabulary without the logits (ops.linear_cross_entropy): refusals and shapes without a GPU, results against the definition in 64 bits on one.

Tolerances, element by element, u = 2^-23 (twice the rounding of a 32-bit operation, since the order of the 16 products inside a matrix instruction is its own):
  logits     products of 16-bit numbers are exact; D of them are added 16 at a time: ez = (D / 16 + 32) u (|x| . |w|).  fp32: an element goes as three parts, exactly, six products for
             one, six times as many additions; the three that are left out are below 2^-24 of the product together, which the 32 u cover.
  loss       twice the largest ez of the row (its log-sum-exp and its own logit), exp and log of 32 bits (16 u (1 + |log-sum-exp|)), and the rounding to the type
  d          a softmax value p is off by p (2 ez + 16 u (1 + |log-sum-exp|)); d = g (p - [target]) is rounded to the type, eps / 2 of it, or to the step 2^-25 below the
             type's normal numbers, under a factor that brings the largest |g| to 2^14 at least; fp32: no rounding, but values below 2^-125 of the largest |g| may be
             taken for zero; the sums over blocks of 16 of it as above
             (u of what was added, or of 2^-126, below which fp32 has steps of 2^-149)
  gradients  that times |w| (or |x|), summed, and the last rounding to the type, of a value or of the smallest normal number"""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lookahead_keys_attention_amd import ops

DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -23
gpu = pytest.mark.gpu


def reference(x, w, target, reduction, dloss, ignore, dtype):
    """(loss, dx, dw) and how far each may be off, in 64 bits on the tensors' device."""
    x, w = x.double(), w.double()
    D, keep = x.shape[1], target != ignore
    half = torch.finfo(dtype).eps / 2
    xk, t = x[keep], target[keep]
    z = xk @ w.T
    ez = (D / 16 + 32) * U * (6 if dtype is torch.float32 else 1) * (xk.abs() @ w.abs().T)
    lse = torch.logsumexp(z, 1, keepdim=True)
    r = torch.arange(len(t), device=x.device)
    loss_k = (lse[:, 0] - z[r, t])
    off_k = 2 * ez.amax(1) + 16 * U * (1 + lse[:, 0].abs())
    p = torch.exp(z - lse)
    n = max(1, len(t))
    g = dloss.double().expand(len(target))[keep] / (n if reduction == "mean" else 1)
    off_p = p * (2 * ez + 16 * U * (1 + lse.abs()))
    p[r, t] -= 1
    d = g[:, None] * p
    most = g.abs().max().item() if len(t) else 0.0
    off_d = g.abs()[:, None] * off_p + (0 if dtype is torch.float32 else half) * d.abs() + {torch.float16: 2.0 ** -25 / 2.0 ** 14, torch.float32: 2.0 ** -125}.get(dtype, 0) * most
    del z, ez, p, off_p
    w_a, x_a, d_a = w.abs(), xk.abs(), d.abs()
    V, six = w.shape[0], 6 if dtype is torch.float32 else 1
    dx_k, off_dx = d @ w, off_d @ w_a + (V / 16 + 32) * U * six * (d_a @ w_a + 2.0 ** -126)
    dw, off_dw = d.T @ xk, off_d.T @ x_a + (n / 16 + 32) * U * six * (d_a.T @ x_a + 2.0 ** -126)
    dx, bound_dx = torch.zeros_like(x), torch.zeros_like(x)
    dx[keep], bound_dx[keep] = dx_k, off_dx
    if reduction == "none":
        loss, bound = torch.zeros(len(target), dtype=torch.float64, device=x.device), torch.zeros(len(target), dtype=torch.float64, device=x.device)
        loss[keep], bound[keep] = loss_k, off_k
    else:   # added in 32 bits by sixteens and then all
        scale = 1 / n if reduction == "mean" else 1
        loss = loss_k.sum() * scale if len(t) or reduction == "sum" else torch.tensor(float("nan"), device=x.device)
        bound = (off_k.sum() + 64 * U * loss_k.abs().sum()) * scale
    return [(loss, bound), (dx, bound_dx), (dw, off_dw)]


def within(got, ref, bound, dtype, what):
    got, half = got.double(), torch.finfo(dtype).eps / 2
    assert got.shape == ref.shape and torch.equal(got.isnan(), ref.isnan()), what
    got, ref = torch.where(ref.isnan(), 0.0, got), torch.where(ref.isnan(), 0.0, ref)
    over = ref.abs() + bound > torch.finfo(dtype).max * (1 - half)   # (rounded to infinity, or not)
    most = bound + half * (ref.abs() + bound).clamp(min=torch.finfo(dtype).tiny)
    off = torch.where(over, 0.0, (got - ref).abs())
    assert (off <= most).all(), (what, (off / most).max())


def inputs(R, V, D, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g) * spread * D ** -0.5
    target = torch.randint(0, V, (R,), generator=g)
    x = torch.randn(R, D, generator=g) + 3 * torch.rand(R, 1, generator=g) * w[target]
    return x.to(dtype).to(DEV), w.to(dtype).to(DEV), target.to(DEV)


def check(x, w, target, reduction="mean", ignore=-100, dloss=None, tell=""):
    dtype = x.dtype
    if dloss is None:
        dloss = torch.tensor(1.25, dtype=dtype, device=DEV) if reduction != "none" else (torch.arange(len(target), device=DEV) % 7 / 4 - 0.5).to(dtype)
    leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    loss = ops.linear_cross_entropy(*leaves, target, reduction, ignore)
    grads = torch.autograd.grad(loss, leaves, dloss)
    for name, got, (ref, bound) in zip(("loss", "dx", "dweight"), (loss.detach(), *grads), reference(x, w, target, reduction, dloss, ignore, dtype)):
        within(got, ref, bound, dtype, (tell, name))
    with torch.no_grad():
        assert torch.equal(ops.linear_cross_entropy(x, w, target, reduction, ignore), loss) or loss.isnan().any()
    return loss, grads


# ---- without a GPU --------------------------------------------------------------------------------------------------
def test_it_traces_and_keeps_shapes():
    with FakeTensorMode():
        x, w = torch.empty(2, 3, 16, dtype=torch.bfloat16, requires_grad=True), torch.empty(50, 16, dtype=torch.bfloat16, requires_grad=True)
        t = torch.zeros(2, 3, dtype=torch.long)
        for reduction, shape in (("mean", ()), ("sum", ()), ("none", (2, 3))):
            x.grad = w.grad = None
            loss = ops.linear_cross_entropy(x, w, t, reduction)
            assert loss.shape == shape and loss.dtype == torch.bfloat16
            loss.sum().backward()
            assert x.grad.shape == x.shape and w.grad.shape == w.shape
        grad, = torch.autograd.grad(ops.linear_cross_entropy(x, w, t).float().square(), w, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            grad.sum().backward()
    for name in ("linear_cross_entropy", "linear_cross_entropy_bwd"):
        assert "!" not in str(getattr(torch.ops.castle_hip, name).default._schema)   # functional


def test_what_it_refuses_without_a_gpu():
    x, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.linear_cross_entropy(x, w, t)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(x, w, t, reduction="median")


def test_entry_points_check_their_arguments_on_the_host():
    from lookahead_keys_attention_amd import _native as N

    lib, i, i64, vp = N.lib(), ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
    state, size = lib.castle_linear_cross_entropy_state_bytes, lib.castle_linear_cross_entropy_workspace_bytes
    state.restype, state.argtypes, size.restype, size.argtypes = i64, [i] * 3, i64, [i] * 5
    assert state(0, 8, 1) == state((1 << 24) + 1, 8, 1) == state(5, 12, 1) == -2 and state(5, 8, 3) == -1
    for rows in (1, 64, 1000):   # what the operator's shape propagation says
        for width in (8, 64, 72):
            for code, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
                _, fake = ops._fake_linear_cross_entropy(torch.empty(rows, width, dtype=dtype), torch.empty(5, width, dtype=dtype), torch.empty(rows, dtype=torch.long), 0, -100)
                assert state(rows, width, code) == fake.numel()
    assert size(5, 10, 8, 3, 0) == -1 and size(5, 10, 8, 1, 4) == size(5, 10, 8, 1, -1) == -5
    for bad in ((0, 10, 8), (5, 0, 8), (5, 10, 0), (5, 10, 12), ((1 << 24) + 1, 10, 8), (5, (1 << 22) + 1, 8), (5, 10, (1 << 16) + 8)):
        assert size(*bad, 1, 0) == -2
    # what the logits would take is not among it: a forward pass of 16 bits holds a copy of the rows and two numbers for each 128 columns, a backward pass about 1 GB of them
    R, V, D = 65536, 131072, 512
    assert size(R, V, D, 1, 0) < 2 * R * D + 8 * R * V // 128 + (4 << 20) < 2 * R * V // 10
    assert size(R, V, D, 1, 3) < 2 * R * D + 4 * 4 * R * D + (1100 << 20) < 2 * R * V // 8
    p = 4096
    fwd = lib.castle_linear_cross_entropy
    fwd.argtypes = [vp, i64, vp, i64, vp, i64, i64, i64, i, i, i, i, vp, vp, i64, i, vp, i64, vp]
    good = [p, 8, p, 8, p, 6, 6, -100, 6, 10, 8, 0, p, p, 1 << 20, 1, p, 1 << 24, None]
    wrong = [(15, 4, -1), (8, 0, -2), (9, 0, -2), (10, 4, -2), (5, 4, -2), (5, 0, -2), (0, None, -5), (0, p + 8, -5), (2, p + 2, -5), (4, p + 4, -5), (1, 12, -5), (3, 12, -5),
             (1, -8, -5), (6, -1, -5), (3, 1 << 23, -5), (11, 3, -5), (11, -1, -5), (12, p + 1, -5), (12, None, -5), (13, None, -4), (13, p + 16, -4), (14, 100, -4), (16, None, -4), (16, p + 64, -4),
             (17, 100, -4)]
    for at, bad, code in wrong:
        args = list(good)
        args[at] = bad
        assert fwd(*args) == code, (at, bad)
    bwd = lib.castle_linear_cross_entropy_bwd
    bwd.argtypes = [vp, i64, vp, i64, vp, i64, i64, i64, i, i, i, i, vp, vp, i64, vp, vp, i, vp, i64, vp]
    good = [p, 8, p, 8, p, 6, 6, -100, 6, 10, 8, 0, p, p, 1 << 20, p, p, 1, p, 1 << 24, None]
    for at, bad, code in wrong[1:18] + [(17, 4, -1), (12, None, -5), (12, p + 1, -5), (15, p + 8, -5), (16, p + 8, -5), (13, None, -4), (14, 100, -4), (18, None, -4), (19, 100, -4)]:
        args = list(good)
        args[at] = bad
        assert bwd(*args) == code, (at, bad)
    good[15] = good[16] = None
    assert bwd(*good) == -5


# ---- on a GPU -------------------------------------------------------------------------------------------------------
# one row, tiles of 64 and 256 rows and their edges; one class, edges of tiles of columns, odd vocabularies; widths below, at and above a step of the contraction
@gpu
@pytest.mark.parametrize("R,V,D", [(1, 1, 8), (1, 2, 64), (3, 255, 16), (63, 256, 56), (64, 257, 64), (65, 1000, 72), (255, 511, 128), (256, 513, 136), (257, 5003, 256),
                                   (700, 300, 512), (1030, 1027, 520), (2, 32000, 512), (300, 50257, 64), (5000, 130, 24)])
@pytest.mark.parametrize("dtype", TYPES)
def test_loss_and_gradients(R, V, D, dtype):
    x, w, target = inputs(R, V, D, dtype, R + V)
    for reduction in ("mean", "sum", "none"):
        check(x, w, target, reduction, tell=reduction)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count(dtype):
    """Any of them, none left, and whatever they hold; another class that does not count; the first class is one like any other."""
    inf, nan = float("inf"), float("nan")
    R, V, D = 200, 300, 72
    x, w, target = inputs(R, V, D, dtype, 5)
    for left in ([], [0], [199], [63, 64], list(range(0, 200, 3)), list(range(65))):
        t = torch.full_like(target, -100)
        t[left] = target[left]
        xb = x.clone()
        gone = t == -100
        xb[gone] = torch.tensor([nan, inf, -inf, torch.finfo(dtype).max, -torch.finfo(dtype).max], device=DEV, dtype=dtype).repeat(D)[:D]
        for reduction in ("mean", "sum", "none"):
            dloss = torch.full((R,), nan, device=DEV, dtype=dtype) if reduction == "none" else torch.tensor(0.5, device=DEV, dtype=dtype)
            if reduction == "none":
                dloss[~gone] = 2
            clean = torch.where(gone[:, None], torch.zeros_like(xb), xb)
            leaves = [xb.requires_grad_(), w.detach().requires_grad_()]
            loss = ops.linear_cross_entropy(*leaves, t, reduction)
            grads = torch.autograd.grad(loss, leaves, dloss)
            assert all(g.isfinite().all() for g in grads) and not grads[0][gone].any() and (left or not grads[1].any())
            ref = reference(clean, w, t, reduction, torch.where(gone, 0, dloss) if reduction == "none" else dloss, -100, dtype)
            for got, (r, bound), what in zip((loss.detach(), *grads), ref, ("loss", "dx", "dw")):
                within(got, r, bound, dtype, (reduction, len(left), what))
    check(x, w, target % 4, ignore=0)
    check(x, w, target % 4, "none", ignore=2)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_classes_that_are_not_there_and_values_that_are_not_numbers(dtype):
    x, w, target = inputs(70, 100, 64, dtype, 6)
    for bad in (100, -1, 1 << 40, -(1 << 40), (1 << 32) + 3):
        t = target.clone()
        t[7] = bad
        leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
        each = ops.linear_cross_entropy(*leaves, t, "none")
        assert each[7].isnan() and each.isnan().sum() == 1
        dx, dw = torch.autograd.grad(each, leaves, torch.ones_like(each))
        assert dx[7].isnan().all() and dx.isnan().any(1).sum() == 1 and dw.isnan().all()
        assert ops.linear_cross_entropy(*leaves, t).isnan()
    for value in (float("nan"), float("inf")):
        xb = x.clone()
        xb[3, 5] = value
        each = ops.linear_cross_entropy(xb, w, target, "none")
        assert each[3].isnan() and each.isnan().sum() == 1
    # a row before which nothing stands but -inf, for one class: all of the rest has no weight
    wb = torch.zeros_like(w)
    wb[:, 0] = -1
    wb[40] = 0
    xb = torch.zeros_like(x)
    xb[:, 0] = float("inf")
    # (inf * 0 of class 40 is a NaN as well)
    assert ops.linear_cross_entropy(xb, wb, torch.full_like(target, 40), "none").isnan().all()
    # logits far from zero, one class alone
    xb = torch.zeros_like(x)
    xb[:, 0] = 200
    check(xb, wb, torch.full_like(target, 40))
    check(xb, wb, torch.full_like(target, 41))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_small_and_large_gradients_of_the_loss(dtype):
    """A mean over many rows, scaled losses: what is multiplied lies in the type's normal numbers whatever the factor."""
    x, w, target = inputs(600, 400, 64, dtype, 8)
    for scale in (2.0 ** -14, 1.0, 2.0 ** 14) + ((2.0 ** -100, 2.0 ** 100) if dtype is not torch.float16 else ()):
        check(x, w, target, "sum", dloss=torch.tensor(scale, dtype=dtype, device=DEV), tell=scale)
        check(x, w, target, "mean", dloss=torch.tensor(scale, dtype=dtype, device=DEV), tell=scale)
    zero = check(x, w, target, dloss=torch.tensor(0.0, dtype=dtype, device=DEV))[1]
    assert not any(g.any() for g in zero)


@gpu
def test_fp32_keeps_what_is_far_below_the_largest():
    """Rows, classes and columns of very different sizes, rows whose losses count very differently, and classes that are as good as impossible: each gradient is as exact as its own sums."""
    g = torch.Generator().manual_seed(17)

    def power(low, high, n):
        return 2.0 ** torch.randint(low, high + 1, (n,), generator=g).float()

    R, V, D = 150, 700, 96
    x, w, target = (t.cpu() for t in inputs(R, V, D, torch.float32, 17, spread=1.0))
    channels = power(-30, 30, D)
    for rows, classes in ((power(-40, 2, R), torch.ones(V)), (torch.ones(R), power(-40, 2, V)), (power(3, 5, R), power(-20, 1, V))):
        xs, ws = (x * rows[:, None] * channels).to(DEV), (w * classes[:, None] / channels).to(DEV)
        check(xs, ws, target.to(DEV))
        check(xs, ws, target.to(DEV), "none", dloss=power(-60, 20, R).to(DEV))
    # a class of softmax values below 2^-60 in every row: its gradient is not zero, and right
    ws = w.clone()
    ws[5] = 0
    xs = x + 64 * torch.eye(D)[0]
    ws[:, 0] = 1
    ws[5, 0] = 0
    _, (_, dw) = check(xs.to(DEV), ws.to(DEV), (target.clamp(min=6)).to(DEV))
    assert 0 < dw[5].abs().max() < 2.0 ** -60
    # the largest numbers of the type as elements: logits beyond it, and far below
    xs, ws = x.clone(), w.clone()
    xs[:, 0], ws[:, 0] = 2.0 ** -130, torch.finfo(torch.float32).max * (1 - 2 * (torch.arange(V) % 2))
    check(xs.to(DEV), ws.to(DEV), target.to(DEV), tell="largest")


@gpu
def test_vocabulary_in_several_pieces():
    """More logits than a workspace holds: 2 and 3 pieces, the last one short and odd."""
    for R, V, dtype in ((4100, 140001, torch.bfloat16), (9000, 131072 + 77, torch.float16), (3000, 100003, torch.float32)):
        x, w, target = inputs(R, V, 16, dtype, R)
        target[::5] = -100
        for reduction in ("mean", "none"):
            check(x, w, target, reduction, tell=(R, reduction))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_and_what_is_asked_for(dtype):
    g = torch.Generator().manual_seed(9)
    wide, table = torch.randn(4, 30, 100, generator=g).to(dtype).to(DEV), (torch.randn(90, 80, generator=g) / 8).to(dtype).to(DEV)
    ids = torch.randint(0, 90, (4, 31), generator=g).to(DEV)
    want = ops.linear_cross_entropy(wide[..., 8:72].contiguous(), table[:, :64].contiguous(), ids[:, 1:].contiguous(), "none")
    for x in (wide[..., 8:72], wide[..., 8:72].contiguous(), wide.transpose(0, 1)[..., 8:72].contiguous().transpose(0, 1)):
        for w in (table[:, :64], table[:, :64].contiguous(), table[:, :64].t().contiguous().t()):
            for t in (ids[:, 1:], ids[:, 1:].int(), ids[:, 1:].t().contiguous().t()):
                assert torch.equal(ops.linear_cross_entropy(x, w, t, "none"), want)
    x, w, t = wide[..., 8:72], table[:, :64], ids[:, 1:]
    both = [x.detach().requires_grad_(), w.detach().requires_grad_()]
    dx, dw = torch.autograd.grad(ops.linear_cross_entropy(*both, t), both)
    assert dx.shape == x.shape and dw.shape == w.shape
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(both[0], w, t), both[0])[0], dx)
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(x, both[1], t), both[1])[0], dw)
    one = ops.linear_cross_entropy(x[0, 0], w, t[0, 0])
    assert one.shape == () and torch.equal(one, want[0, 0])
    for shape in ((0, 64), (2, 0, 64)):
        x0 = torch.zeros(shape, dtype=dtype, device=DEV, requires_grad=True)
        t0 = torch.zeros(shape[:-1], dtype=torch.long, device=DEV)
        assert ops.linear_cross_entropy(x0, both[1], t0).isnan() and ops.linear_cross_entropy(x0, both[1], t0, "sum") == 0
        assert ops.linear_cross_entropy(x0, both[1], t0, "none").shape == t0.shape
        d = torch.autograd.grad(ops.linear_cross_entropy(x0, both[1], t0, "sum"), (x0, both[1]))
        assert d[0].shape == shape and not d[1].any()
    for bad in (lambda: ops.linear_cross_entropy(x, w, t.cpu()), lambda: ops.linear_cross_entropy(x, w.double(), t), lambda: ops.linear_cross_entropy(x, w[:, :32], t),
                lambda: ops.linear_cross_entropy(x, w, t[:, 1:]), lambda: ops.linear_cross_entropy(x, w, t.float()), lambda: ops.linear_cross_entropy(x[..., :20], w[:, :20], t),
                lambda: ops.linear_cross_entropy(x, w[:0], t), lambda: ops.linear_cross_entropy(x.double(), w.double(), t)):
        with pytest.raises((TypeError, ValueError)):
            bad()


@gpu
def test_gradients_against_differences():
    """In fp32: the change of the loss along a direction, against the gradients, with a step whose errors of second order and of rounding are both below 1 % of it."""
    x, w, target = inputs(50, 120, 32, torch.float32, 11)
    g = torch.Generator().manual_seed(1)
    dx, dw = (torch.randn(t.shape, generator=g).to(DEV) for t in (x, w))
    leaves = [x.requires_grad_(), w.requires_grad_()]
    gx, gw = torch.autograd.grad(ops.linear_cross_entropy(*leaves, target), leaves)
    with torch.no_grad():
        for ax, aw in ((1, 0), (0, 1), (1, 1)):
            h = 2.0 ** -6
            up, down = (ops.linear_cross_entropy(x + s * h * ax * dx, w + s * h * aw * dw, target).double() for s in (1, -1))
            slope = (ax * (gx * dx).double().sum() + aw * (gw * dw).double().sum())
            assert abs((up - down) / (2 * h) - slope) <= 0.01 * (gx.norm() * dx.norm() * ax + gw.norm() * dw.norm() * aw) / 8


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_same_every_time_in_graphs_and_on_other_streams(dtype):
    x, w, target = inputs(300, 1000, 64, dtype, 12)
    target[::4] = -100
    leaves = [x.requires_grad_(), w.requires_grad_()]
    one = torch.ones((), dtype=dtype, device=DEV)

    def step():
        loss = ops.linear_cross_entropy(*leaves, target)
        return loss.detach(), *torch.autograd.grad(loss, leaves, one)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):   # (other rows count each time)
        target.copy_(torch.where(torch.arange(300, device=DEV) % (k + 2) == 0, -100, torch.arange(300, device=DEV)))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


@gpu
def test_rows_past_32_bits_of_elements():
    """Hidden rows of more than 2^32 elements: the last ones have a loss, a gradient and a part in the weight's."""
    R, D, V, few, dtype = 65600, 65536, 40, 30, torch.bfloat16
    g = torch.Generator().manual_seed(14)
    x = torch.zeros(R, D, dtype=dtype, device=DEV)
    x[-few:] = torch.randn(few, D, generator=g).to(dtype).to(DEV)
    w = (torch.randn(V, D, generator=g) * D ** -0.5).to(dtype).to(DEV)
    target = torch.randint(0, V, (R,), generator=g).to(DEV)
    dloss = torch.zeros(R, dtype=dtype, device=DEV)
    dloss[-few:] = 0.75
    leaves = [x.requires_grad_(), w.requires_grad_()]
    each = ops.linear_cross_entropy(*leaves, target, "none")
    dx, dw = torch.autograd.grad(each, leaves, dloss)
    ref = reference(x[-few:].detach(), w.detach(), target[-few:], "none", dloss[-few:], -100, dtype)
    for got, (r, bound), what in zip((each[-few:].detach(), dx[-few:], dw), ref, ("loss", "dx", "dw")):
        within(got, r, bound, dtype, what)
    assert not dx[:-few].any()


@gpu
def test_a_vocabulary_past_32_bits_of_elements():
    """Rows of zeros but for the last ones: their logits are 0, their softmax values one number of each row."""
    R, D, V, few, dtype = 5, 65536, 65600, 30, torch.bfloat16
    g = torch.Generator().manual_seed(15)
    x = torch.randn(R, D, generator=g).to(dtype).to(DEV)
    w = torch.zeros(V, D, dtype=dtype, device=DEV)
    w[-few:] = (torch.randn(few, D, generator=g) * D ** -0.5).to(dtype).to(DEV)
    target = torch.tensor([V - 1, V - 30, V - 31, 0, V - 2], device=DEV)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    each = ops.linear_cross_entropy(*leaves, target, "none")
    dx, dw = torch.autograd.grad(each, leaves, torch.ones_like(each))
    z = torch.zeros(R, V, dtype=torch.float64, device=DEV)
    z[:, -few:] = x.detach().double() @ w[-few:].detach().double().T
    d = torch.softmax(z, 1)
    d[range(R), target] -= 1
    # as for the other sizes: logits off by ez, softmax values by 2 ez, d and the result by half a step
    x64, w64 = x.detach().double(), w[-few:].detach().double()
    ez = (D / 16 + 32) * U * (x64.abs() @ w64.abs().T).max()
    for got, ref, most in ((each.detach(), torch.logsumexp(z, 1) - z[range(R), target], 1.0), (dx, d[:, -few:] @ w64, d[:, -few:].abs() @ w64.abs()),
                           (dw[-few:], d[:, -few:].T @ x64, d[:, -few:].T.abs() @ x64.abs()), (dw[:3], d[:, :3].T @ x64, d[:, :3].T.abs() @ x64.abs()),
                           (dw[32768:32771], d[:, 32768:32771].T @ x64, d[:, 32768:32771].T.abs() @ x64.abs())):
        assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (1.02 * 2.0 ** -8 + 2 * ez) * most).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_calls_that_run_at_once(dtype):
    """Two streams with inputs of their own, and a leaf and a gradient of the loss that are not at 16 bytes."""
    calls = [inputs(500 + 100 * k, 700, 64, dtype, 16 + k) for k in range(2)]
    want = [check(*c)[1] for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for k, (x, w, target) in enumerate(calls):
            with torch.cuda.stream(streams[k]):
                leaves = [x.detach().requires_grad_(), w.detach().requires_grad_()]
                got[k] = torch.autograd.grad(ops.linear_cross_entropy(*leaves, target), leaves, torch.tensor(1.25, dtype=dtype, device=DEV))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    x, w, target = calls[0]
    odd = torch.cat((x.new_zeros(1), x.flatten()))[1:].view(x.shape)
    dloss = torch.arange(1, len(target) + 2, device=DEV).to(dtype)[1:]
    leaves = [odd.requires_grad_(), w.requires_grad_()]
    a = torch.autograd.grad(ops.linear_cross_entropy(*leaves, target, "none"), leaves, dloss)
    leaves[0] = x.detach().requires_grad_()
    b = torch.autograd.grad(ops.linear_cross_entropy(*leaves, target, "none"), leaves, dloss.clone())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@gpu
def test_opcheck():
    x, w, target = inputs(20, 30, 16, torch.float32, 13)
    torch.library.opcheck(torch.ops.castle_hip.linear_cross_entropy.default, (x.requires_grad_(), w.requires_grad_(), target, 0, -100),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
