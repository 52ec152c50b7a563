"""Norms on both sides of a residual sum (ops.residual_norm): refusals and shapes without a GPU, results against the formula in 64 bits on one.

Tolerances.  u = 2^-24 is the rounding of a 32-bit operation.  The mean of D squares is added up by lanes, D / 8 additions one behind the other at most, so a norm's factor is off by (D / 8 + 12) u / 2 + 4 u at most;
with c = (D + 64) u for everything that stands before a result, each of them is off by c times the sum of the magnitudes of what it is made of.  A column sum of R rows adds R u of its magnitudes.
The last rounding is half a step of the type."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lookahead_keys_attention_amd import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
U = 2.0 ** -24
EPS = torch.finfo(torch.float32).eps
NAMES = ("x", "residual", "weight", "scale", "gate", "next_weight")


def inputs(shape, dtype, gate=None, without=(), seed=0):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    n = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(dtype)
    t = {"x": n(*shape, std=0.5), "residual": n(*shape, std=2), "weight": n(D, std=0.2, mean=1), "scale": n(D, std=0.1, mean=0.3),
         "gate": None if gate is None else torch.rand(*gate, generator=g).to(dtype), "next_weight": n(D, std=0.2, mean=1)}
    for name in without:
        t[name] = None
    return t, n(*shape), n(*shape)


def reference(t, dy, dh, eps=EPS):
    """{name: (value, sum of magnitudes)} in 64 bits; dy or dh may be None."""
    shape = t["x"].shape
    D = shape[-1]
    d = {k: None if v is None else v.double() for k, v in t.items()}
    one = torch.ones((), dtype=torch.float64)
    x, r = d["x"], d["residual"]
    w, s, g, nw = (one if d[k] is None else d[k] for k in NAMES[2:])
    inv = (x.square().mean(-1, keepdim=True) + eps).rsqrt() if d["weight"] is not None else one
    xh = x * inv
    c = w * s
    q = c * g * xh
    y = r + q
    out = {"y": (y, r.abs() + q.abs())}
    inv_y = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    yh = y * inv_y
    yh_off = (r.abs() + q.abs()) * inv_y
    if d["next_weight"] is not None:
        out["h"] = (yh * nw, yh_off * nw.abs())
    if dy is None and dh is None:
        return out
    dt, dt_off = torch.zeros_like(x), torch.zeros_like(x)
    if dy is not None:
        dt, dt_off = dt + dy.double(), dt_off + dy.double().abs()
    if dh is not None:
        dn = dh.double() * nw
        dt = dt + inv_y * (dn - yh * (dn * yh).mean(-1, keepdim=True))
        dt_off = dt_off + inv_y * (dn.abs() + 2 * yh_off * (dn.abs() * yh_off).mean(-1, keepdim=True))
        out["next_weight"] = ((dh.double() * yh).reshape(-1, D).sum(0), (dh.double().abs() * yh_off).reshape(-1, D).sum(0))
    else:
        out["next_weight"] = (torch.zeros(D, dtype=torch.float64),) * 2
    e, e_off = dt * c * g, dt_off * (c * g).abs()
    if d["weight"] is not None:
        out["x"] = (inv * (e - xh * (e * xh).mean(-1, keepdim=True)), inv * (e_off + 2 * xh.abs() * (e_off * xh.abs()).mean(-1, keepdim=True)))
    else:
        out["x"] = (e, e_off)
    out["residual"] = (dt, dt_off)
    p, p_off = dt * xh, dt_off * xh.abs()
    rows = lambda v: v.expand(shape).reshape(-1, D).sum(0)
    out["weight"] = (rows(p * g * s), rows(p_off * (g * s).abs()))
    out["scale"] = (rows(p * g * w), rows(p_off * (g * w).abs()))
    if d["gate"] is not None:
        like = d["gate"].shape if d["gate"].dim() == len(shape) else (1,) * (len(shape) - 1) + (D,)
        out["gate"] = ((p * c).sum_to_size(like).reshape(d["gate"].shape), (p_off * c.abs()).sum_to_size(like).reshape(d["gate"].shape))
    return out


def within(got, ref, rows, D, dtype, what):
    value, magnitude = ref
    got = got.detach().cpu().double()
    assert got.shape == value.shape and got.isfinite().all(), what
    slack = (D + 64 + rows) * U * magnitude
    most = slack + torch.finfo(dtype).eps / 2 * (value.abs() + slack).clamp(min=torch.finfo(dtype).tiny)
    worst = ((got - value).abs() - most).max() if got.numel() else 0.0
    assert worst <= 0, (what, float(worst))


def call(leaves):
    return ops.residual_norm(leaves["x"], leaves["residual"], **{k: leaves[k] for k in NAMES[2:]})


def check(t, dy, dh, dtype, use=(True, True)):
    rows, D = t["x"].numel() // t["x"].shape[-1], t["x"].shape[-1]
    dy, dh = dy if use[0] else None, dh if use[1] and t["next_weight"] is not None else None
    ref = reference(t, dy, dh)
    leaves = {k: None if v is None else v.to(DEV).requires_grad_() for k, v in t.items()}
    out = call(leaves)
    y, h = out if t["next_weight"] is not None else (out, None)
    within(y, ref["y"], 0, D, dtype, "y")
    if h is not None:
        within(h, ref["h"], 0, D, dtype, "h")
    there = {k: v for k, v in leaves.items() if v is not None}
    outputs = [(o, d.to(DEV)) for o, d in ((y, dy), (h, dh)) if d is not None]
    grads = torch.autograd.grad([o for o, _ in outputs], list(there.values()), [d for _, d in outputs], allow_unused=True)
    for name, got in zip(there, grads):
        within(got, ref[name], rows if name in NAMES[2:] else 0, D, dtype, name)


# ---- without a GPU --------------------------------------------------------------------------------------------------
def test_traces_and_keeps_shapes():
    with FakeTensorMode():
        x, r, gate = (torch.empty(*s, dtype=torch.bfloat16, requires_grad=True) for s in ((2, 3, 20), (2, 3, 20), (2, 1, 20)))
        w = torch.empty(20, dtype=torch.bfloat16, requires_grad=True)
        y, h = ops.residual_norm(x, r, weight=w, gate=gate, next_weight=w)
        assert y.shape == h.shape == x.shape and h.dtype == torch.bfloat16
        (y.sum() + h.sum()).backward()
        assert x.grad.shape == r.grad.shape == x.shape and gate.grad.shape == gate.shape and w.grad.shape == w.shape
        assert ops.residual_norm(x, r).shape == x.shape


@pytest.mark.parametrize("change", [
    dict(residual=torch.zeros(2, 3, 8)), dict(weight=torch.zeros(8)), dict(scale=torch.zeros(1, 16)), dict(next_weight=torch.zeros(16, dtype=torch.float16)),
    dict(gate=torch.zeros(1, 3, 16)), dict(gate=torch.zeros(3, 16)), dict(gate=torch.zeros(2, 3, 1)), dict(eps=-1.0), dict(),
])
def test_refusals_on_the_host(change):
    args = dict(x=torch.zeros(2, 3, 16), residual=torch.zeros(2, 3, 16)) | change
    with pytest.raises((ValueError, RuntimeError)):
        ops.residual_norm(**args)


# ---- on a GPU -------------------------------------------------------------------------------------------------------
WIDTHS = [1, 7, 8, 100, 128, 200, 256, 257, 512, 1000, 1024, 1500, 2048, 2056, 4096, 5001, 8192]


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", WIDTHS)
def test_values_and_gradients(D, dtype):
    for rows, gate in ((1, None), (5, "full"), (33, None), (34, "pairs")):
        shape = (rows, D) if gate != "pairs" else (2, 17, D)
        check(*inputs(shape, dtype, None if gate is None else shape if gate == "full" else (2, 1, D), seed=rows), dtype)


@gpu
@pytest.mark.parametrize("shape, gate", [
    ((3, 700, 64), (3, 1, 64)), ((1, 3000, 40), (1, 1, 40)), ((40, 3, 136), (40, 1, 136)), ((2, 5, 7, 24), (2, 5, 1, 24)), ((2, 5, 7, 24), (2, 1, 1, 24)), ((2, 5, 7, 24), (1, 1, 1, 24)),
    ((9, 24), (24,)), ((6, 11, 24), (24,)), ((6, 1, 24), (6, 1, 24)), ((5000, 1, 16), (1, 1, 16)), ((300, 9, 1200), (300, 1, 1200)), ((24,), (24,)), ((70, 300, 8), (70, 1, 8)),
])
def test_gates_of_several_rows(shape, gate):
    for dtype in (torch.bfloat16, torch.float32):
        check(*inputs(shape, dtype, gate), dtype)


@gpu
@pytest.mark.parametrize("without", [(), ("weight",), ("scale",), ("next_weight",), ("weight", "scale"), ("weight", "next_weight"), ("weight", "scale", "next_weight")])
@pytest.mark.parametrize("gate", [None, (3, 1, 72), (3, 50, 72)])
def test_parts_that_are_left_out(without, gate):
    for use in ((True, True), (True, False), (False, True)):
        if use == (False, True) and "next_weight" in without:
            continue
        check(*inputs((3, 50, 72), torch.bfloat16, gate, without), torch.bfloat16, use)


@gpu
def test_many_rows_and_those_of_large_and_small_size():
    t, dy, dh = inputs((20000, 24), torch.float32)
    t["x"][::3] *= 1e12    # (squares of which reach 1e24; a norm's factor is 1e-12)
    t["x"][1::3] *= 1e-12   # (below the eps of the norm)
    check(t, dy, dh, torch.float32)
    t["x"][4], t["residual"][4] = 0, 0
    check(t, dy, dh, torch.float32)


@gpu
@pytest.mark.parametrize("need", range(1, 64, 5))
def test_gradients_that_are_asked_for(need):
    t, dy, dh = inputs((4, 9, 72), torch.bfloat16, (4, 1, 72))
    ref = reference(t, dy, dh)
    leaves = {k: v.to(DEV).requires_grad_(bool(need >> i & 1)) for i, (k, v) in enumerate(t.items())}
    y, h = call(leaves)
    torch.autograd.backward((y, h), (dy.to(DEV), dh.to(DEV)))
    for i, (k, leaf) in enumerate(leaves.items()):
        if need >> i & 1:
            within(leaf.grad, ref[k], 36, 72, torch.bfloat16, k)
        else:
            assert leaf.grad is None


@gpu
def test_strides_and_alignment():
    for dtype in (torch.bfloat16, torch.float32):
        t, dy, dh = inputs((3, 11, 72), dtype, (3, 1, 72))
        want = call({k: v.to(DEV) for k, v in t.items()})
        odd = lambda v: torch.cat((v.flatten(), v.new_zeros(1))).to(DEV).roll(1)[1:].view(v.shape)
        turned = lambda v: v.transpose(0, -1).contiguous().to(DEV).transpose(0, -1)
        for f in (odd, turned):
            got = call({k: f(v) for k, v in t.items()})
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        wide = torch.zeros(3, 11, 80, dtype=dtype, device=DEV)
        wide[..., :72] = t["x"].to(DEV)
        got = call({k: wide[..., :72] if k == "x" else v.to(DEV) for k, v in t.items()})
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_what_is_not_finite_stays_in_its_row_and_rows_of_zeros():
    t, dy, dh = inputs((40, 96), torch.bfloat16)
    clean = call({k: v.to(DEV) if v is not None else None for k, v in t.items()})
    t["x"][3, 5], t["residual"][9, 0] = float("inf"), float("nan")
    t["x"][11], t["residual"][11] = 0, 0
    y, h = call({k: v.to(DEV) if v is not None else None for k, v in t.items()})
    keep = [r for r in range(40) if r not in (3, 9, 11)]
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(h[keep], clean[1][keep])
    assert h[9].isnan().all() and h[3].isnan().any() and not y[11].any() and not h[11].any()


@gpu
def test_empty_calls():
    t, dy, dh = inputs((0, 16), torch.bfloat16)
    leaves = {k: v.to(DEV).requires_grad_() if v is not None else None for k, v in t.items()}
    y, h = call(leaves)
    assert y.shape == h.shape == (0, 16)
    torch.autograd.backward((y, h), (dy.to(DEV), dh.to(DEV)))
    assert not leaves["weight"].grad.any() and leaves["x"].grad.shape == (0, 16)


@gpu
def test_the_same_bits_every_time_on_any_stream_and_in_a_graph():
    t, dy, dh = inputs((6, 500, 200), torch.bfloat16, (6, 1, 200))
    leaves = {k: v.to(DEV).requires_grad_() for k, v in t.items()}
    dy, dh = dy.to(DEV), dh.to(DEV)

    def step():
        y, h = call(leaves)
        return (y.detach(), h.detach(), *torch.autograd.grad((y, h), list(leaves.values()), (dy, dh)))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        with torch.no_grad():
            leaves["x"].copy_(t["x"].to(DEV) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), k


@gpu
def test_refusals_on_the_gpu():
    t, dy, dh = inputs((4, 64), torch.bfloat16)
    g = {k: v.to(DEV) if v is not None else None for k, v in t.items()}
    for change in (dict(weight=g["weight"].float()), dict(scale=g["scale"].cpu()), dict(x=torch.zeros(4, 8193, device=DEV), residual=torch.zeros(4, 8193, device=DEV))):
        with pytest.raises((ValueError, RuntimeError)):
            call(g | change)
    with pytest.raises((TypeError, RuntimeError)):
        ops.residual_norm(g["x"].double(), g["residual"].double())
    w = g["weight"].clone().requires_grad_()
    dw, = torch.autograd.grad(call(g | dict(weight=w))[0], w, dy.to(DEV), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dw.sum().backward()


@gpu
def test_a_recorded_backward_pass_beside_one_that_lives_is_refused():
    x, r, w = (torch.randn(4, 64, device=DEV, requires_grad=True), torch.randn(4, 64, device=DEV, requires_grad=True), torch.ones(64, device=DEV, requires_grad=True))
    kept = ops.residual_norm(x, r, weight=w, next_weight=w)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(ops.residual_norm(x, r, weight=w, next_weight=w)[1].sum(), (x, r, w))
    torch.cuda.synchronize()
    want = [t.clone() for t in torch.autograd.grad(kept[1].sum(), (x, r, w))]
    del kept
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(ops.residual_norm(x, r, weight=w, next_weight=w)[1].sum(), (x, r, w))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


@pytest.mark.parametrize("change, error, what", [
    (dict(residual=torch.zeros(2, 3, 8)), ValueError, "one shape"), (dict(residual=torch.zeros(1, 3, 16)), ValueError, "one shape"), (dict(x=torch.zeros(()), residual=torch.zeros(())), ValueError, "one shape"),
    (dict(weight=torch.zeros(8)), ValueError, "columns"), (dict(scale=torch.zeros(1, 16)), ValueError, "columns"), (dict(next_weight=torch.zeros(17)), ValueError, "columns"),
    (dict(next_weight=torch.zeros(16, dtype=torch.float16)), ValueError, "one type"), (dict(gate=torch.zeros(2, 3, 16).half()), ValueError, "one type"),
    (dict(residual=torch.zeros(2, 3, 16).half()), ValueError, "one type"),
    (dict(gate=torch.zeros(1, 3, 16)), ValueError, "gate"), (dict(gate=torch.zeros(3, 16)), ValueError, "gate"), (dict(gate=torch.zeros(2, 3, 1)), ValueError, "gate"),
    (dict(gate=torch.zeros(3, 1, 16)), ValueError, "gate"), (dict(gate=torch.zeros(8)), ValueError, "gate"),
    (dict(eps=-1.0), ValueError, "eps"), (dict(eps=float("nan")), ValueError, "eps"),
    (dict(x=torch.zeros(2, 8193), residual=torch.zeros(2, 8193)), ValueError, "8192"), (dict(x=torch.zeros(2, 0), residual=torch.zeros(2, 0)), ValueError, "8192"),
    (dict(x=torch.zeros(2, 16).double(), residual=torch.zeros(2, 16).double()), TypeError, "double|Double|float64"),
    (dict(), RuntimeError, "on the GPU"),
])
def test_each_refusal_by_its_message(change, error, what):
    """What is wrong with the sizes is said of tensors on the CPU too."""
    args = dict(x=torch.zeros(2, 3, 16), residual=torch.zeros(2, 3, 16)) | change
    with pytest.raises(error, match=what) as refused:
        ops.residual_norm(**args)
    assert type(refused.value) is error


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [24, 200, 700, 1500, 3000, 6000])
@pytest.mark.parametrize("gate", [None, "each", "shared"])
def test_gradients_do_not_meet_what_they_do_not_depend_on(gate, D, dtype):
    """Without a norm behind the block the gradients of x and of the residual are those of finite numbers whatever x and the residual hold, as those of x are with one whatever the residual holds and those of the residual
    whatever x holds; rows of zeros as gradients have zeros as theirs."""
    shape = (3, 4, D)
    bad = [float("inf"), float("nan"), -float("inf")]
    for without in (("weight", "next_weight"), ("next_weight",), ("weight",), ()):
        t, dy, _ = inputs(shape, dtype, {None: None, "each": shape, "shared": (3, 1, D)}[gate], without)
        dy = dy.to(DEV)
        dy[2, 1] = 0

        def grads(change):
            leaves = {k: None if v is None else v.to(DEV).clone() for k, v in t.items()}
            for name in change:
                for i, b in enumerate(bad):
                    leaves[name][i, 1, 5 * i] = b
            leaves = {k: None if v is None else v.requires_grad_() for k, v in leaves.items()}
            out = call(leaves)
            y = out if torch.is_tensor(out) else out[0]   # (no gradient of the norm in front of the next block)
            return torch.autograd.grad(y, (leaves["x"], leaves["residual"]), dy)

        clean = grads(())
        for change in (("residual",),) if t["weight"] is not None else (("residual",), ("x",), ("x", "residual")):
            for a, b, name in zip(grads(change), clean, ("x", "residual")):
                assert torch.equal(a, b), (without, change, name)
        assert torch.equal(grads(("x",))[1], dy) and torch.equal(clean[1], dy) and not clean[0][2, 1].any()
