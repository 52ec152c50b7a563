"""Gated feed-forward block (ops.gated_feed_forward): refusals and shapes without a GPU, results against the formula in 64 bits on one.

Tolerances, from the formula with every error that the kernels may make.  E = 2^-23 is what an addition of a matrix product may lose (2^-24 rounded, twice that cut off), H half a step of the
type.  A hidden sum of n products of exact 16-bit numbers (fp32: of three parts, 2^-22 more) is off by (n + 8) E of the sum of its magnitudes.  act moves by 1.13 of what its argument does, its
slope by 0.8; both are evaluated to 2^-18 of themselves (gelu: 3e-6 where it counts), and next to zero to 2^-24.  In 16 bits a = act(g) and b = v act'(g) lose what lies below 24 bits, 2^-16,
h, dg and dv are rounded once, H.  Each product adds up what its operands are off by and its own sum's error, and the result is rounded: H."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lookahead_keys_attention_amd import GatedFeedForward, _native, ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
E = 2.0 ** -23


def inputs(R, D, F, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    return [t.to(dtype) for t in (n(R, D) * spread, n(2 * F, D) * D ** -0.5, n(D, F) * F ** -0.5, n(R, D))]


def act_of(g, activation):
    """act, its slope"""
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    cdf = 0.5 * torch.erfc(-g * 0.5 ** 0.5)
    return g * cdf, cdf + g * torch.exp(-g * g / 2) * 0.3989422804014327


def few(R, D, F):
    """Sizes where what the roundings of h, dg and dv leave takes part in the products."""
    return min(R * D, D * F, R * F) < 4096


def reference(x, win, wout, dy, activation, dtype):
    """{name: (value, what the result may be off by before it is rounded)} in 64 bits."""
    H = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    keep = 1.0   # how much of a rounding of h, dg and dv counts; in two parts that of the second one, and float16 ends at 2^-25
    least = 0.0
    if H and few(x.shape[0], x.shape[1], wout.shape[1]):
        keep, least = H, 2.0 ** -25 if dtype == torch.float16 else 0.0
    more = 2.0 ** -22 if dtype == torch.float32 else 0.0
    x, win, wout, dy = (t.double() for t in (x, win, wout, dy))
    R, D, F = x.shape[0], x.shape[1], wout.shape[1]

    def product(a, b, da, db):
        """a b and its error, of operands that are off by da and db (or exact)"""
        off = ((a.shape[1] + 8) * E + more) * (a.abs() @ b.abs())
        if da is not None:
            off = off + da @ b.abs()
        if db is not None:
            off = off + a.abs() @ db
        return a @ b, off

    u, du_off = product(x, win.T, None, None)
    g, v = u.chunk(2, 1)
    g_off, v_off = du_off.chunk(2, 1)
    act, slope = act_of(g, activation)
    act_off = 1.13 * g_off + 2.0 ** -18 * act.abs() + 2.0 ** -24
    slope_off = 0.8 * g_off + 2.0 ** -18 * slope.abs() + 2.0 ** -24
    h = act * v
    h_off = act_off * v.abs() + act.abs() * v_off + act_off * v_off + H * keep * h.abs() + least + (2.0 ** -24 * h.abs())
    y = product(h, wout.T, h_off, None)
    dh, dh_off = product(dy, wout, None, None)
    cut = 2.0 ** -16 if H else 2.0 ** -23
    a_off, b = act_off + cut * act.abs(), v * slope
    b_off = slope_off * v.abs() + slope.abs() * v_off + slope_off * v_off + cut * b.abs()
    d = torch.cat((dh * b, dh * act), 1)
    d_off = torch.cat((dh_off * (b.abs() + b_off) + dh.abs() * b_off, dh_off * (act.abs() + a_off) + dh.abs() * a_off), 1)
    d_off = d_off + (H * keep + 2.0 ** -23) * (d.abs() + d_off) + least
    return {"y": y, "dx": product(d, win, d_off, None), "dwin": product(d.T, x, d_off.T, None), "dwout": product(dy.T, h, None, h_off)}


def within(got, ref, dtype, what):
    value, off = ref
    got = got.detach().cpu().double()
    most = off + torch.finfo(dtype).eps / 2 * (value.abs() + off).clamp(min=torch.finfo(dtype).tiny)
    assert got.shape == value.shape, what
    assert got.isfinite().all(), what
    worst = ((got - value).abs() - most).max() if got.numel() else 0.0
    assert worst <= 0, (what, float(worst))


def run(x, win, wout, dy, activation):
    leaves = [t.to(DEV).requires_grad_() for t in (x, win, wout)]
    y = ops.gated_feed_forward(*leaves, activation=activation)
    grads = torch.autograd.grad(y, leaves, dy.to(DEV))
    return dict(zip(("y", "dx", "dwin", "dwout"), (y, *grads)))


# ---- without a GPU --------------------------------------------------------------------------------------------------
def test_traces_and_keeps_shapes():
    with FakeTensorMode():
        for dtype in (torch.bfloat16, torch.float32):
            x, win, wout = (torch.empty(*s, dtype=dtype, requires_grad=True) for s in ((2, 3, 16), (80, 16), (16, 40)))
            y = ops.gated_feed_forward(x, win, wout)
            assert y.shape == x.shape and y.dtype == dtype
            y.sum().backward()
            assert all(t.grad.shape == t.shape for t in (x, win, wout))


@pytest.mark.parametrize("change, error", [
    (dict(x=torch.zeros(2, 12)), ValueError),                                    # another width
    (dict(win=torch.zeros(24, 16)), ValueError),                                 # not twice the hidden width
    (dict(x=torch.zeros(2, 12), win=torch.zeros(32, 12), wout=torch.zeros(12, 16)), ValueError),   # widths of no whole pieces
    (dict(wout=torch.zeros(16, 16, dtype=torch.bfloat16)), ValueError),
    (dict(activation="relu"), ValueError),
    (dict(), RuntimeError),                                                      # tensors on the CPU
])
def test_refusals_on_the_host(change, error):
    args = dict(x=torch.zeros(2, 16), win=torch.zeros(32, 16), wout=torch.zeros(16, 16), activation="silu") | change
    with pytest.raises((error, RuntimeError)):
        ops.gated_feed_forward(args["x"], args["win"], args["wout"], activation=args["activation"])


# ---- on a GPU -------------------------------------------------------------------------------------------------------
SIZES = [(1, 8, 8), (3, 64, 128), (64, 72, 136), (65, 136, 40), (200, 512, 680), (513, 256, 264), (129, 1024, 128)]


@gpu
@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("R, D, F", SIZES)
def test_values_and_gradients(R, D, F, dtype, activation):
    t = inputs(R, D, F, dtype, seed=R)
    ref = reference(*t, activation, dtype)
    for name, got in run(*t, activation).items():
        within(got, ref[name], dtype, name)


# one, two and four rows of waves to a tile; tiles that end inside in both directions; a contraction that ends inside a step
@gpu
@pytest.mark.parametrize("R, D, F", [(4090, 64, 1016), (8190, 64, 1016), (8200, 200, 1032), (300, 1000, 2048)])
def test_sizes_of_tiles(R, D, F):
    t = inputs(R, D, F, torch.bfloat16, seed=1)
    t_gpu = [x.to(DEV) for x in t]   # (the reference of these sizes is formed on the GPU)
    ref = {k: (v.cpu(), off.cpu()) for k, (v, off) in reference(*t_gpu, "silu", torch.bfloat16).items()}
    for name, got in run(*t, "silu").items():
        within(got, ref[name], torch.bfloat16, name)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R, D, F", [(199, 1024, 4096), (3000, 768, 2048), (12345, 200, 520), (1000, 2048, 4096), (2048, 2048, 3000), (8192, 512, 1408), (12345, 512, 1400), (9999, 256, 1000)])
def test_weight_gradients_of_one_launch(R, D, F, dtype):
    """Tiles taken whole, in ranges, both, with the input gradient among them; contractions that end inside a step, with rows behind the end that are not finite; ragged tiles; the same bits again."""
    x, win, wout, dy = (t.to(DEV) for t in inputs(R, D, F, dtype, seed=R))
    ref = {k: (v.cpu(), off.cpu()) for k, (v, off) in reference(x, win, wout, dy, "silu", dtype).items()}
    longer = [torch.cat((t, torch.full((64, D), float("nan"), device=DEV, dtype=dtype))) for t in (x, dy)]
    x, dy = (t[:R] for t in longer)
    got = run(x, win, wout, dy, "silu")
    for k in ref:
        within(got[k], ref[k], dtype, k)
    again = run(x, win, wout, dy, "silu")
    assert all(torch.equal(got[k], again[k]) for k in got)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R, D, F", [(2048, 64, 64), (3000, 64, 128), (4096, 128, 320), (777, 768, 2048), (128, 768, 768), (100, 2048, 72)])
def test_gradients_of_one_launch(R, D, F, dtype):
    """All three products of the backward pass together, in ranges of the rows or not, and the two launches where a third does not fit."""
    t = inputs(R, D, F, dtype, seed=R + F)
    ref = {k: (v.cpu(), off.cpu()) for k, (v, off) in reference(*(x.to(DEV) for x in t), "silu", dtype).items()}
    got, again = run(*t, "silu"), run(*t, "silu")
    for name in ref:
        within(got[name], ref[name], dtype, name)
        assert torch.equal(got[name], again[name])
    with torch.no_grad():   # (fp32: the gate on the product's store, or where the product goes in ranges by itself)
        y = ops.gated_feed_forward(*(x.to(DEV) for x in t[:3]))
    within(y, ref["y"], dtype, "y without gradients")


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 2, 16, 17, 32, 50, 64])
def test_tokens_without_gradients(rows, dtype):
    for D, F in ((64, 24), (512, 1408), (1040, 72)):
        x, win, wout, dy = inputs(rows, D, F, dtype, seed=rows)
        with torch.no_grad():
            y = ops.gated_feed_forward(*(t.to(DEV) for t in (x[:, None], win, wout)))
        within(y[:, 0], reference(x, win, wout, dy, "silu", dtype)["y"], dtype, (D, F))


@gpu
@pytest.mark.parametrize("need", range(1, 8))
def test_gradients_that_are_asked_for(need):
    for dtype in (torch.bfloat16, torch.float32):
        t = inputs(70, 64, 72, dtype)
        ref = reference(*t, "silu", dtype)
        leaves = [x.to(DEV).requires_grad_(bool(need >> i & 1)) for i, x in enumerate(t[:3])]
        y = ops.gated_feed_forward(*leaves)
        y.backward(t[3].to(DEV))
        for i, (leaf, name) in enumerate(zip(leaves, ("dx", "dwin", "dwout"))):
            if need >> i & 1:
                within(leaf.grad, ref[name], dtype, name)
            else:
                assert leaf.grad is None


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R, D, F", [(1, 2048, 1408), (8, 24, 192), (2, 64, 584), (33, 64, 56), (70, 40, 1024), (255, 16, 24), (5770, 16, 24), (70000, 8, 8), (40, 96, 4000)])
def test_few_numbers_are_rounded_once(R, D, F, dtype):
    """As far from the formula as results rounded once, but for sums in 32 bits and a and b in 24 bits (2^-13 of half a step): 1.02 times.  (Each row of long contractions too.)"""
    assert few(R, D, F)
    t = inputs(R, D, F, dtype, seed=R)
    ref = reference(*(x.to(DEV) for x in t), "gelu", dtype)
    got = run(*t, "gelu")
    for name, (value, off) in ref.items():
        within(got[name], (value.cpu(), off.cpu()), dtype, name)
        once, here = (value.to(dtype).double() - value).norm(), (got[name].detach().double() - value).norm()
        assert here <= 1.02 * once, (name, float(here / once))
    with torch.no_grad():
        y = ops.gated_feed_forward(*(x.to(DEV) for x in t[:3]), activation="gelu")
    value = ref["y"][0]
    assert (y.double() - value).norm() <= 1.02 * (value.to(dtype).double() - value).norm()


@gpu
def test_strides_of_all_operands():
    for dtype in (torch.bfloat16, torch.float32):
        x, win, wout, dy = inputs(40, 64, 72, dtype)
        ref = reference(x, win, wout, dy, "silu", dtype)
        wide = lambda t: torch.cat((t, t.new_full((t.shape[0], 24), float("nan"))), 1).to(DEV)[:, :t.shape[1]]   # rows apart
        turned = lambda t: t.t().contiguous().to(DEV).t()                                                        # columns apart
        odd = lambda t: torch.cat((t.flatten(), t.new_zeros(1))).to(DEV).roll(1)[1:].view(t.shape)               # not 16-byte aligned
        for f in (wide, turned, odd):
            leaves = [f(t).detach().requires_grad_() for t in (x, win, wout)]
            y = ops.gated_feed_forward(*leaves)
            grads = torch.autograd.grad(y, leaves, f(dy))
            for name, got in zip(("y", "dx", "dwin", "dwout"), (y, *grads)):
                within(got, ref[name], dtype, name)


@gpu
@pytest.mark.parametrize("R, D, F, dtype", [(8, 24, 192, torch.bfloat16), (300, 200, 520, torch.bfloat16), (199, 1024, 4096, torch.bfloat16), (12345, 512, 1400, torch.bfloat16), (300, 200, 520, torch.float32),
                                            (100, 2048, 72, torch.float32)])
def test_rows_apart_and_some_of_the_gradients(R, D, F, dtype):
    """Every way that the backward pass goes: rows of all operands with NaNs between them, and each choice of gradients, which are those of all three."""
    t = inputs(R, D, F, dtype, seed=R)
    ref = {k: (v.cpu(), off.cpu()) for k, (v, off) in reference(*(x.to(DEV) for x in t), "silu", dtype).items()}
    apart = [torch.cat((x, x.new_full((x.shape[0], 40), float("nan"))), 1).to(DEV)[:, :x.shape[1]] for x in t]
    for need in range(1, 8):
        leaves = [x.detach().requires_grad_(bool(need >> i & 1)) for i, x in enumerate(apart[:3])]
        y = ops.gated_feed_forward(*leaves)
        asked = [(leaf, name) for leaf, name in zip(leaves, ("dx", "dwin", "dwout")) if leaf.requires_grad]
        for got, (_, name) in zip(torch.autograd.grad(y, [leaf for leaf, _ in asked], apart[3]), asked):
            within(got, ref[name], dtype, (name, need))
        within(y, ref["y"], dtype, "y")


@gpu
def test_shapes_and_empty_calls():
    x, win, wout, dy = (t.to(DEV) for t in inputs(24, 64, 72, torch.bfloat16))
    flat = ops.gated_feed_forward(x, win, wout)
    assert torch.equal(ops.gated_feed_forward(x.view(2, 3, 4, 64), win, wout).view(24, 64), flat)
    assert torch.equal(ops.gated_feed_forward(x[0], win, wout), ops.gated_feed_forward(x[:1], win, wout)[0])
    leaves = [t.clone().requires_grad_() for t in (x[:0], win, wout)]
    y = ops.gated_feed_forward(*leaves)
    assert y.shape == (0, 64)
    y.backward(dy[:0])
    assert leaves[0].grad.shape == (0, 64) and not leaves[1].grad.any() and not leaves[2].grad.any()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_far_arguments_and_what_is_not_finite(dtype):
    """Gates of +-1000 are one and zero; a NaN or an infinity of a row stays in that row.  (Not in fp16, which ends at 65504: hidden numbers are 1000 times 1000 here, and infinite in it.)"""
    D, F = 64, 72
    x, win, wout, dy = inputs(66, D, F, dtype, spread=1000.0)
    ref = reference(x, win, wout, dy, "silu", dtype)
    for name, got in run(x, win, wout, dy, "silu").items():
        within(got, ref[name], dtype, name)
    ref = reference(x, win, wout, dy, "gelu", dtype)
    x[5, 3], x[7, 60] = float("nan"), float("inf")
    bad = run(x, win, wout, dy, "gelu")
    keep = [r for r in range(66) if r not in (5, 7)]
    for name in ("y", "dx"):
        # (not the same bits in fp32: a tile of a product in which something is not finite goes to other instructions)
        within(bad[name][keep], tuple(t[keep] for t in ref[name]), dtype, name)
        assert bad[name][5].isnan().all(), name


@gpu
def test_the_same_bits_every_time_on_any_stream_and_in_a_graph():
    t = [x.to(DEV) for x in inputs(700, 136, 264, torch.bfloat16)]
    leaves = [x.clone().requires_grad_() for x in t[:3]]

    def step():
        y = ops.gated_feed_forward(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, t[3]))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(t[0] * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), k


@gpu
@pytest.mark.parametrize("R, D, F", [(3000, 768, 2048), (300, 64, 136), (6, 40, 1024)])
def test_two_streams_at_once_and_a_graph(R, D, F):
    """Weight gradients in whole tiles and ranges, in the launch of all three, in two parts: calls of two streams side by side, and replays among eager calls."""
    sets = [[t.to(DEV) for t in inputs(R, D, F, torch.bfloat16, seed=k)] for k in range(2)]
    want = [{k: v.detach() for k, v in run(*t, "gelu").items()} for t in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(5):
        for t, stream, g in zip(sets, streams, got):
            with torch.cuda.stream(stream):
                g.append({k: v.detach() for k, v in run(*t, "gelu").items()})   # (no pass is kept alive: see below)
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(r[k], w[k]) for r in g for k in w)
    x, win, wout, dy = [t.detach().clone() for t in sets[0]]
    leaves = [t.requires_grad_() for t in (x, win, wout)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.gated_feed_forward(*leaves, activation="gelu")
        grads = torch.autograd.grad(y, leaves, dy)
    for k in (1, 0, 1):
        with torch.no_grad():
            for t, new in zip((x, win, wout, dy), sets[k]):
                t.copy_(new)
        graph.replay()
        other = run(*sets[1 - k], "gelu")
        torch.cuda.synchronize()
        assert all(torch.equal(a, want[k][name]) for a, name in zip((y, *grads), ("y", "dx", "dwin", "dwout")))
        assert all(torch.equal(other[name], want[1 - k][name]) for name in other)


@gpu
@pytest.mark.parametrize("leaves_of_its_own", [True, False])
def test_a_recorded_backward_pass_beside_one_that_lives_is_refused(leaves_of_its_own):
    x, win, wout, dy = (t.to(DEV) for t in inputs(64, 64, 128, torch.bfloat16))
    leaves = [t.requires_grad_() for t in (x, win, wout)]
    kept = ops.gated_feed_forward(*leaves)
    inside = leaves if leaves_of_its_own else [t.clone() for t in leaves]   # (or what an earlier pass would reach)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(ops.gated_feed_forward(*inside), inside, dy)
    torch.cuda.synchronize()
    want = [t.clone() for t in torch.autograd.grad(kept, leaves, dy)]
    del kept, inside
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(ops.gated_feed_forward(*leaves), leaves, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


@gpu
def test_refusals_on_the_gpu():
    x, win, wout, dy = (t.to(DEV) for t in inputs(4, 64, 72, torch.bfloat16))
    with pytest.raises(ValueError):
        ops.gated_feed_forward(x, win.float(), wout)
    with pytest.raises(ValueError):
        ops.gated_feed_forward(x, win.cpu(), wout)
    with pytest.raises((TypeError, RuntimeError)):
        ops.gated_feed_forward(x.double(), win.double(), wout.double())
    big = torch.empty(1, dtype=torch.bfloat16, device=DEV).expand(1 << 24, 64)   # hidden rows of 2^24 x 144 elements
    with pytest.raises(ValueError):
        ops.gated_feed_forward(big, win, wout)
    w = win.clone().requires_grad_()
    y = ops.gated_feed_forward(x, w, wout)
    dw, = torch.autograd.grad(y, w, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dw.sum().backward()
    y = ops.gated_feed_forward(x, w, wout)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1000, 40000, 80000, 131072, 190000])
def test_traced_states_of_more_than_two_gigabytes(rows, dtype):
    with FakeTensorMode():
        x, win, wout = (torch.empty(*s, dtype=dtype) for s in ((rows, 64), (2 * 5504, 64), (64, 5504)))
        state = torch.ops.castle_hip.gated_feed_forward(x, win, wout, 0, True)[1].numel()
    least = 8 * rows * 5504   # u; or h and 6 bytes of a and b
    assert least <= state <= 1.03 * least + (1 << 20)


def test_limits_of_the_block_are_those_of_the_operator():
    """`gated_sizes_ok` says what castle_gated_state_bytes does, on both sides of every limit."""
    last = (1 << 31) // (2 * 5504) - 192   # rows of which (rows + 192) 2 F is about 2^31
    sizes = [(r, 64, 5504) for r in range(last - 1, last + 3)] + [((1 << 31) // 4096 - 192 + k, 4096, 64) for k in (-1, 0, 1)]
    sizes += [(8, 1 << 20, 1024 - 96 + 8 * k) for k in range(-2, 3)] + [(8, 1024, (1 << 20) + 8 * k) for k in (-1, 0, 1)] + [(8, 2048 - 192 + 8 * k, 1 << 20) for k in (-1, 0, 1)]
    sizes += [(8, 12, 8), (8, 8, 12), (8, 0, 8), (8, 8, 0), (1, 8, 8), (1 << 31, 8, 8), ((1 << 27) - 192, 16, 8), ((1 << 27) - 193, 16, 8)]
    seen = set()
    for rows, dim, hidden in sizes:
        ok = _native.lib().castle_gated_state_bytes(rows, dim, hidden, 1) > 0 if rows < 1 << 31 else False
        assert ops.gated_sizes_ok(rows, dim, hidden) == ok, (rows, dim, hidden)
        seen.add(ok)
    assert seen == {True, False} and ops.gated_sizes_ok(0, 8, 8)


@gpu
def test_module_over_more_rows_than_the_operator_takes():
    """The formulation, whose rows are those of the operator over fewer."""
    block = GatedFeedForward(8, 5504).to(DEV, torch.bfloat16)
    rows = (1 << 31) // (2 * 5504)
    x = torch.randn(rows, 8, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.gated_feed_forward(x, block.to_hidden.weight, block.to_out.weight)
    with torch.no_grad():
        y, part = block(x), block(x[-500:])
    assert y.shape == x.shape
    off = (y[-500:].float() - part.float()).abs().max() / part.float().abs().max()
    assert off < 2.0 ** -6   # the formulation rounds both halves, the gate, and what it times: 4 half steps of bf16, and the result


@pytest.mark.parametrize("change, error, what", [
    (dict(x=torch.zeros(2, 24)), ValueError, "x is"),                            # another width
    (dict(win=torch.zeros(24, 16)), ValueError, "x is"),                         # not twice the hidden width
    (dict(wout=torch.zeros(8, 16)), ValueError, "x is"),
    (dict(win=torch.zeros(32, 16, 1)), ValueError, "x is"),
    (dict(x=torch.zeros(())), ValueError, "x is"),
    (dict(x=torch.zeros(2, 12), win=torch.zeros(32, 12), wout=torch.zeros(12, 16)), ValueError, "multiples of 8"),
    (dict(win=torch.zeros(24, 16), wout=torch.zeros(16, 12)), ValueError, "multiples of 8"),
    (dict(win=torch.zeros(0, 16), wout=torch.zeros(16, 0)), ValueError, "multiples of 8"),
    (dict(x=torch.zeros(2, 0), win=torch.zeros(32, 0), wout=torch.zeros(0, 16)), ValueError, "multiples of 8"),
    (dict(wout=torch.zeros(16, 16, dtype=torch.bfloat16)), ValueError, "one type"),
    (dict(x=torch.zeros(1, 16).expand(1 << 27, 16)), ValueError, "less than 2\\^31 elements"),
    (dict(x=torch.zeros(2, 16, dtype=torch.float64), win=torch.zeros(32, 16, dtype=torch.float64), wout=torch.zeros(16, 16, dtype=torch.float64)), TypeError, "float64|double|Double"),
    (dict(), RuntimeError, "on the GPU"),
])
def test_each_refusal_by_its_message(change, error, what):
    """What is wrong with the sizes is said of tensors on the CPU too."""
    args = dict(x=torch.zeros(2, 16), win=torch.zeros(32, 16), wout=torch.zeros(16, 16)) | change
    with pytest.raises(error, match=what) as refused:
        ops.gated_feed_forward(args["x"], args["win"], args["wout"])
    assert type(refused.value) is error


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R, D, F", [(3, 64, 72), (33, 64, 56), (40, 24, 200), (300, 16, 24), (70, 64, 72)])
def test_infinities_of_weights_and_gradients(R, D, F, dtype):
    """An infinite weight or gradient meets what the rounding of a hidden number has left, zero where nothing has: results are infinite where the formula's are, and NaN where those are."""
    x, win, wout, dy = inputs(R, D, F, dtype, seed=R)
    wout[3, 5], dy[1, 7] = float("inf"), -float("inf")
    for changed in ((x, win, wout, dy.clamp(-3, 3)), (x, win, wout.clamp(-3, 3), dy)):
        got = run(*changed, "silu")
        with torch.no_grad():
            got["y of tokens"] = ops.gated_feed_forward(*(t.to(DEV) for t in changed[:3]))
        a, b, c, d = (t.double() for t in changed)
        g, v = (a @ b.T).chunk(2, 1)
        act, slope = act_of(g, "silu")
        h, dh = act * v, d @ c
        du = torch.cat((dh * (v * slope), dh * act), 1)
        want = {"y": h @ c.T, "y of tokens": h @ c.T, "dx": du @ b, "dwin": du.T @ a, "dwout": d.T @ h}
        for name, value in want.items():
            here = got[name].detach().cpu().double()
            assert torch.equal(here.isnan(), value.isnan()), name
            assert torch.equal(here.isinf(), value.isinf()) and torch.equal(here[here.isinf()], value[value.isinf()]), name
