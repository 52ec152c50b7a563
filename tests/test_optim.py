"""AdamW over many tensors (ops.adamw_step, ops.gradient_norm, AdamW): refusals without a GPU, results against the formula in 64 bits on one.

Tolerances.  u = 2^-24 is the rounding of a 32-bit operation.  Moments: two products and a sum, 4 u of their magnitudes (with the factor of clipping, itself 4 u, 8 u).  A parameter: its decay 2 u, its step about 12 u
of the step, and where sums cancel of their magnitudes.  What is rounded by chance lies between the two neighbours of the number before: within one step of the type, 2^-3 of an e4m3 number (2^-9 of 448 below its
normal numbers), eps of a 16-bit one; and its mean over many draws is the number itself, within 6 of the mean's standard deviations, at most half a step each over the root of their number."""
import copy
import io
import math
import pickle

import pytest
import torch

from lookahead_keys_attention_amd import AdamW, ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
U = 2.0 ** -24
OPTIONS = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def tensors(shapes, dtype, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dtype).to(device) for s in shapes]


def formula(p, g, m, v, t, clip=1.0, lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05):
    """(p, m, v, magnitude of p's parts, of its step) in 64 bits."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * clip
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    step = lr / (1 - betas[0] ** t) * m / ((v / (1 - betas[1] ** t)).sqrt() + eps)
    return p * (1 - lr * weight_decay) - step, m, v, p.abs() + step.abs()


def close(got, want, most, what):
    off = (got.detach().cpu().double() - want).abs()
    assert got.shape == want.shape and (off <= most).all(), (what, float((off - most).max()))


def blocks_of(x):
    """x in rows of 256, zeros behind its end"""
    n = x.numel()
    return torch.cat((x.flatten(), x.new_zeros(-n % 256))).view(-1, 256)


def values(codes, exponents):
    """what states of 8 bits stand for, in 64 bits, in their order"""
    x = codes.cpu().float().double()
    return (blocks_of(x) * torch.exp2(exponents.cpu().double())[:, None]).flatten()[:x.numel()]


def empty_states(shapes, bits, device=DEV):
    if bits == 32:
        return [torch.zeros(s, device=device) for s in shapes], [torch.zeros(s, device=device) for s in shapes], None, None
    zero = lambda s: torch.zeros(s, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    exponents = lambda s: torch.zeros((math.prod(s) + 255) // 256, dtype=torch.int8, device=device)
    return [zero(s) for s in shapes], [zero(s) for s in shapes], [exponents(s) for s in shapes], [exponents(s) for s in shapes]


def seed_of(n=12345):
    return torch.tensor([n], device=DEV)


def counter(n=0):
    return torch.tensor([n], device=DEV)


# ---- without a GPU --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("options", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_norm=-1.0), dict(state_bits=16),
                                     dict(lr=torch.zeros(2)), dict(lr=torch.zeros(1, dtype=torch.float64))])
def test_options_that_are_refused(options):
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(3))], **options)


def test_parameters_on_the_cpu_are_refused():
    p = torch.nn.Parameter(torch.zeros(3))
    optimizer = AdamW([p])
    assert optimizer.step() is None   # (no gradient yet: nothing to do)
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="GPU"):
        optimizer.step()
    one = torch.zeros(3)
    with pytest.raises(RuntimeError):
        ops.adamw_step([one], [one], [one], [one], torch.zeros(1, dtype=torch.int64), lr=1e-3)
    with pytest.raises(RuntimeError):
        ops.gradient_norm([one])
    with pytest.raises((ValueError, RuntimeError)):
        ops.gradient_norm([])


# ---- on a GPU -------------------------------------------------------------------------------------------------------
SHAPES = [(1,), (7,), (8,), (255,), (256, 3), (2049,), (0, 5), (1000, 33), (64, 64, 5), ()]


@gpu
@pytest.mark.parametrize("clip", [None, 1.0, 1e9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_with_states_of_32_bits(dtype, clip):
    shapes = SHAPES
    params = tensors(shapes, dtype, 1, DEV)
    m, v, _, _ = empty_states(shapes, 32)
    step = counter(4)
    for k in range(3):
        grads = tensors(shapes, dtype, 10 + k, DEV)
        before = [[x.cpu() for x in t] for t in (params, m, v)]
        norm = ops.adamw_step(params, grads, m, v, step, max_norm=clip, **OPTIONS)
        assert int(step) == 5 + k
        factor = 1.0
        if clip is not None:
            exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
            assert abs(float(norm) - exact) <= 2 * U * exact
            factor = min(1.0, clip / (exact + 1e-6))
        else:
            assert norm is None
        for i, g in enumerate(grads):
            p0, m0, v0 = (x[i] for x in before)
            p, m1, v1, size = formula(p0, g.cpu(), m0, v0, 5 + k, factor)
            close(m[i], m1, 8 * U * (m0.double().abs() + g.cpu().double().abs() * factor), "m")
            close(v[i], v1, 16 * U * (v0.double() + (g.cpu().double() * factor) ** 2), "v")
            slack = 40 * U * size + 3e-3 * 40 * U   # (a step is about lr, whatever cancels in m)
            close(params[i], p, slack + torch.finfo(dtype).eps / 2 * (p.abs() + slack).clamp(min=torch.finfo(dtype).tiny) if dtype != torch.float32 else slack, "p")


@gpu
@pytest.mark.parametrize("count", [1, 63, 64, 65, 200])
def test_lists_of_any_length(count):
    """As many tensors one by one."""
    shapes = [((i * 37) % 300 + 1,) for i in range(count)]
    for bits in (32, 8):
        params, grads = tensors(shapes, torch.bfloat16, 1, DEV), tensors(shapes, torch.bfloat16, 2, DEV)
        m, v, em, ev = empty_states(shapes, bits)
        if bits == 32:
            ops.adamw_step(params, grads, m, v, counter(), **OPTIONS)
            for i in range(count):
                p, = tensors(shapes, torch.bfloat16, 1, DEV)[i:i + 1]
                one = empty_states(shapes[i:i + 1], bits)
                ops.adamw_step([p], [grads[i]], one[0], one[1], counter(), **OPTIONS)
                assert torch.equal(p, params[i]) and torch.equal(one[0][0], m[i]) and torch.equal(one[1][0], v[i])
        else:   # (a tensor's number decides its random numbers: the exponents, which have no part in them, are alike)
            ops.adamw_step(params, grads, m, v, counter(), seed=seed_of(), exp_avg_exponents=em, exp_avg_sq_exponents=ev, **OPTIONS)
            for i in range(count):
                one = empty_states(shapes[i:i + 1], bits)
                p = [tensors(shapes, torch.bfloat16, 1, DEV)[i]]
                ops.adamw_step(p, [grads[i]], one[0], one[1], counter(), seed=seed_of(), exp_avg_exponents=one[2], exp_avg_sq_exponents=one[3], **OPTIONS)
                assert torch.equal(one[2][0], em[i]) and torch.equal(one[3][0], ev[i])
                assert i > 0 or torch.equal(p[0], params[0])


def check_chance(got, exponents, want, positive):
    """States of 8 bits against what they are rounded from: the exponent that the largest finite one needs, one of the two neighbours; NaN for what is not finite."""
    finite = want.flatten().isfinite()
    assert torch.equal(got.flatten().cpu().float().isfinite(), finite)
    flat = torch.where(finite, want.flatten(), 0.0)
    top = blocks_of(flat.abs()).amax(1)
    power = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / 448)).clamp(-126, 120)
    near = (top / 448 / torch.exp2(power) - 1).abs() < 1e-5   # (on the border the last bit of 32 decides)
    near |= (top / 448 / torch.exp2(power) - 0.5).abs() < 1e-5
    assert ((exponents.cpu().double() == power) | near | (top == 0)).all()
    scale = torch.exp2(exponents.cpu().double()).repeat_interleave(256)[:flat.numel()]
    x = torch.where(finite, values(got.flatten(), exponents), 0.0)
    step = torch.maximum(torch.exp2(torch.floor(torch.log2(flat.abs().clamp(min=1e-300))) - 3), scale * 2.0 ** -9)
    off = (x - flat).abs()
    assert (off <= step * (1 + 1e-5) + 16 * U * flat.abs()).all(), float((off / step).max())
    if positive:
        assert (x[flat > 0] > 0).all()
    assert (x[flat == 0] == 0).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_with_states_of_8_bits(dtype):
    shapes = SHAPES
    params = tensors(shapes, dtype, 1, DEV)
    m, v, em, ev = empty_states(shapes, 8)
    step = counter()
    for k in range(3):
        grads = tensors(shapes, dtype, 10 + k, DEV)
        for g in grads:   # sizes of many orders, zeros among them
            g.mul_(torch.exp2(-torch.arange(g.numel(), device=DEV) % 23.0).view(g.shape).to(dtype))
            g.view(-1)[::5] = 0
        before = [[x.clone() for x in t] for t in (params, m, v, em, ev)]
        ops.adamw_step(params, grads, m, v, step, seed=seed_of(), exp_avg_exponents=em, exp_avg_sq_exponents=ev, **OPTIONS)
        for i, g in enumerate(grads):
            p0, m0, v0, em0, ev0 = (x[i] for x in before)
            old_m, old_r = values(m0.flatten(), em0), values(v0.flatten(), ev0)
            p, m1, v1, size = formula(p0.cpu().flatten(), g.cpu().flatten(), old_m, old_r * old_r, k + 1)
            check_chance(m[i], em[i], m1, False)
            check_chance(v[i], ev[i], v1.sqrt(), True)
            # a step is about lr at most: |m| is not much larger than the root of v, and the element's own gradient bounds how far the rest is off
            slack = 60 * U * size + 1e-6
            step_of_type = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps * (p.abs() + slack).clamp(min=torch.finfo(dtype).tiny)
            # (in fp16 some gradients of 2^22 and less are infinite: their parameters are not finite either, and stay so)
            finite = p.isfinite()
            assert torch.equal(params[i].flatten().cpu().isfinite(), finite)
            close(params[i].flatten().cpu()[finite], p[finite], (slack + step_of_type)[finite], "p")


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_mean_of_what_is_rounded_by_chance(dtype):
    """65536 parameters of one size take one step; states are those of the first step, which their gradient alone decides."""
    n = 65536
    for value, grad in ((1.0, 0.3), (-3.3e-3, 1.7e-4), (2e-6, -5e-7)):
        p = torch.full((n,), value, dtype=dtype, device=DEV)
        g = torch.full((n,), grad, dtype=dtype, device=DEV)
        g[::256] = grad * 3   # (the largest of each block, so that the others lie between two numbers)
        m, v, em, ev = empty_states([(n,)], 8)
        p0, g0 = p.cpu().clone(), g.cpu()
        ops.adamw_step([p], [g], m, v, counter(), seed=seed_of(7), exp_avg_exponents=em, exp_avg_sq_exponents=ev, **OPTIONS)
        want, m1, v1, _ = formula(p0, g0, torch.zeros(n), torch.zeros(n), 1)
        rest = torch.arange(n) % 256 != 0
        for got, exact in ((p.cpu().double(), want), (values(m[0], em[0]), m1), (values(v[0], ev[0]), v1.sqrt())):
            got, exact = got[rest], exact[rest]
            step = float((got.max() - got.min()))
            assert step > 0 and len(got.unique()) == 2   # two neighbours
            assert abs(float(got.mean() - exact.mean())) <= 6 * step / 2 / math.sqrt(len(got)) + 32 * U * abs(float(exact.mean()))


@gpu
def test_random_numbers_are_those_that_are_described():
    """Philox of the published description, on the host: of one group of eight elements the second moment, the first one and the parameter."""
    from test_tokens import philox

    p = torch.full((2, 8), 1.0, dtype=torch.bfloat16, device=DEV)
    g = torch.full((2, 8), 0.37, dtype=torch.bfloat16, device=DEV)
    (m,), (v,), (em,), (ev,) = empty_states([(2, 8)], 8)
    key, number, step = -987654321, 1, 41
    other = torch.ones(3, dtype=torch.bfloat16, device=DEV)
    states = empty_states([(3,)], 8)
    lists = lambda a, b: [a, b]
    ops.adamw_step(lists(other, p), lists(other.clone(), g), lists(states[0][0], m), lists(states[1][0], v), counter(step - 1), seed=seed_of(key),
                   exp_avg_exponents=lists(states[2][0], em), exp_avg_sq_exponents=lists(states[3][0], ev), **OPTIONS)
    want, m1, v1, _ = formula(torch.ones(1), g.flatten()[:1].cpu(), torch.zeros(1), torch.zeros(1), step)
    for kind, got, exact, spacing, base in ((0, values(v.flatten(), ev), v1.sqrt(), 2.0 ** -3, None), (1, values(m.flatten(), em), m1, 2.0 ** -3, None), (2, p.cpu().double().flatten(), want, 2.0 ** -7, None)):
        x = float(exact)
        size = 2.0 ** math.floor(math.log2(abs(x))) * spacing
        below = math.floor(x / size) * size
        share = (x - below) / size
        for i in range(2):
            words = philox([4 * i + kind], key % 2 ** 64, step | number << 32)[0]
            halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
            for e in range(8):
                if abs(halves[e] / 65536 + share - 1) < 1e-3:
                    continue   # (too near to the border for 64 bits to decide)
                up = halves[e] / 65536 + share >= 1
                assert float(got[8 * i + e]) == pytest.approx(below + size * up, rel=1e-9), (kind, i, e)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_of_gradients(dtype):
    for seed, shapes in enumerate(([(1,)], SHAPES, [(i + 1,) for i in range(130)], [(3_000_001,)])):
        grads = tensors(shapes, dtype, seed, DEV)
        exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        got = ops.gradient_norm(grads)
        assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - exact) <= U * exact
        assert torch.equal(got, ops.gradient_norm(grads))
    if dtype != torch.float16:   # squares beyond 32 bits, both ways
        assert float(ops.gradient_norm([torch.full((100,), 1e30, dtype=dtype, device=DEV)])) == pytest.approx(1e31, rel=2 ** -7)
        assert float(ops.gradient_norm([torch.full((100,), 1e-30, dtype=dtype, device=DEV)])) == pytest.approx(1e-29, rel=2 ** -7)
    bad = torch.ones(5000, dtype=dtype, device=DEV)
    bad[4321] = float("inf")
    assert ops.gradient_norm([bad]).isinf()
    bad[7] = float("nan")
    assert ops.gradient_norm([bad]).isnan()
    assert float(ops.gradient_norm([torch.zeros(0, dtype=dtype, device=DEV)])) == 0
    turned = torch.randn(30, 20, device=DEV).to(dtype)
    assert float(ops.gradient_norm([turned.t()])) == float(ops.gradient_norm([turned]))
    assert float(ops.gradient_norm([turned[:, ::2]])) == pytest.approx(float(turned[:, ::2].double().norm()), rel=1e-6)


@gpu
def test_alignment_layouts_and_gradients_of_other_layouts():
    flat = torch.randn(5000, device=DEV).bfloat16()
    grad = torch.randn(5000, device=DEV).bfloat16()
    for lo in (0, 1, 3, 7):   # pieces of one buffer, at any element
        states = [torch.zeros(5000, device=DEV) for _ in range(2)]
        bytes_ = [torch.zeros(5000, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
        exponents = [torch.zeros(17, dtype=torch.int8, device=DEV) for _ in range(2)]
        part = slice(lo, lo + 4099)
        p1, p2, p3 = flat.clone(), flat[part].clone(), flat.clone()
        ops.adamw_step([p1[part]], [grad[part]], [states[0][part]], [states[1][part]], counter(), **OPTIONS)
        alone = [torch.zeros(4099, device=DEV) for _ in range(2)]
        ops.adamw_step([p2], [grad[part].clone()], [alone[0]], [alone[1]], counter(), **OPTIONS)
        assert torch.equal(p1[part], p2) and torch.equal(states[0][part], alone[0]) and torch.equal(states[1][part], alone[1])
        outside = torch.ones(5000, dtype=torch.bool, device=DEV)
        outside[part] = False
        assert torch.equal(p1[outside], flat[outside]) and not states[0][outside].any()
        ops.adamw_step([p3[part]], [grad[part]], [bytes_[0][part]], [bytes_[1][part]], counter(), seed=seed_of(), exp_avg_exponents=[exponents[0]], exp_avg_sq_exponents=[exponents[1]], **OPTIONS)
        assert torch.equal(p3[outside], flat[outside]) and not bytes_[0].view(torch.uint8)[outside].any() and not bytes_[1].view(torch.uint8)[outside].any()
    a = torch.randn(12, 40, device=DEV)
    g = torch.randn(12, 40, device=DEV)
    p, q = a.clone(), a.t().contiguous().t()   # the same parameter, stored the other way
    sp, sq = [torch.zeros_like(p) for _ in range(2)], [torch.zeros_like(q) for _ in range(2)]
    ops.adamw_step([p], [g.t().contiguous().t()], [sp[0]], [sp[1]], counter(), **OPTIONS)
    ops.adamw_step([q], [g], [sq[0]], [sq[1]], counter(), **OPTIONS)
    assert torch.equal(p, q) and torch.equal(sp[0], sq[0])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_finite_stays_where_it_is(bits):
    for bad in (float("nan"), float("inf")):
        p, g = tensors([(700,)], torch.bfloat16, 1, DEV)[0], tensors([(700,)], torch.bfloat16, 2, DEV)[0]
        g[300] = bad
        m, v, em, ev = empty_states([(700,)], bits)
        step = counter()
        for _ in range(2):
            ops.adamw_step([p], [g], m, v, step, seed=seed_of(), exp_avg_exponents=em, exp_avg_sq_exponents=ev, **OPTIONS)
            g[300] = 1
        there = torch.arange(700, device=DEV) == 300
        assert torch.equal(p.isnan(), there)
        read = (lambda t, e: t[0].float()) if bits == 32 else (lambda t, e: values(t[0], e[0]).to(DEV))
        assert read(m, em)[~there].isfinite().all() and not read(m, em)[there].isfinite().any() and not read(v, ev)[there].isfinite().any()


@gpu
def test_steps_in_a_graph_are_those_outside():
    shapes = [(300,), (64, 40), (5,)]
    for bits, dtype in ((32, torch.float32), (8, torch.bfloat16)):
        def fresh():
            return tensors(shapes, dtype, 1, DEV), empty_states(shapes, bits), counter(), torch.tensor([1e-3], device=DEV)

        grads = tensors(shapes, dtype, 2, DEV)

        def step(params, states, count, lr):
            return ops.adamw_step(params, grads, states[0], states[1], count, lr=lr, max_norm=0.5, seed=seed_if, exp_avg_exponents=states[2], exp_avg_sq_exponents=states[3])

        seed_if = seed_of()
        one, two = fresh(), fresh()
        step(*one), step(*two)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            norm = step(*one)
        for k in range(4):
            for x in (one, two):
                x[3].fill_(1e-3 * (k + 1))
            for g in grads:
                g.mul_(1.5)
            graph.replay()
            want = step(*two)
            torch.cuda.synchronize()
            assert torch.equal(norm, want) and int(one[2]) == int(two[2]) == k + 2
            flat = lambda x: [t.view(torch.uint8) for part in (x[0], *(s for s in x[1] if s is not None)) for t in part]
            assert all(torch.equal(a, b) for a, b in zip(flat(one), flat(two))), k


@gpu
def test_refusals_on_the_gpu():
    p, g = tensors([(300,), (300,)], torch.bfloat16, 1, DEV)
    m, v, em, ev = empty_states([(300,)], 32)
    sm, sv, sem, sev = empty_states([(300,)], 8)
    good = dict(params=[p], grads=[g], exp_avgs=m, exp_avg_sqs=v, step=counter(), lr=1e-3)
    bad = [
        dict(params=[]), dict(grads=[g, g]), dict(grads=[g.float()]), dict(grads=[g[:200]]), dict(exp_avgs=[m[0].double()]), dict(exp_avgs=[m[0].bfloat16()]), dict(exp_avgs=[m[0][:200]]),
        dict(exp_avgs=sm, exp_avg_sqs=sv), dict(step=torch.zeros(1, device=DEV)), dict(step=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(step=torch.zeros(1, dtype=torch.int64)),
        dict(betas=(1.0, 0.5)), dict(eps=-1.0), dict(max_norm=-1.0), dict(weight_decay=-0.1), dict(lr=torch.zeros(1, dtype=torch.float64, device=DEV)), dict(lr=torch.zeros(1)),
        dict(seed=torch.zeros(2, dtype=torch.int64, device=DEV)), dict(exp_avg_exponents=sem), dict(exp_avg_sqs=m),
        dict(exp_avgs=sm, exp_avg_sqs=sv, exp_avg_exponents=sem, exp_avg_sq_exponents=sev),   # no seed
        dict(exp_avgs=sm, exp_avg_sqs=sv, exp_avg_exponents=[sem[0][:1]], exp_avg_sq_exponents=sev, seed=seed_of()),
        dict(params=[p, p], grads=[g, g], exp_avgs=m + [m[0].clone()], exp_avg_sqs=v + [v[0].clone()]),   # the same twice
        dict(params=[p, p[100:200]], grads=[g, g[:100]], exp_avgs=m + [torch.zeros(100, device=DEV)], exp_avg_sqs=v + [torch.zeros(100, device=DEV)]),
        dict(params=[p[::2]], grads=[g[::2]], exp_avgs=[m[0][::2]], exp_avg_sqs=[v[0][::2]]),
        dict(params=[p.expand(2, 300)], grads=[g.expand(2, 300)], exp_avgs=[torch.zeros(2, 300, device=DEV)], exp_avg_sqs=[torch.zeros(2, 300, device=DEV)]),
        dict(params=[p.double()], grads=[g.double()]),
    ]
    before = p.clone()
    for change in bad:
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            ops.adamw_step(**(good | change))
            raise AssertionError(f"accepted: {change.keys()}")
    assert torch.equal(p, before) and not m[0].any()
    ops.adamw_step(**good)
    assert not torch.equal(p, before)


def model(dtype, device=DEV):
    torch.manual_seed(3)
    return torch.nn.Sequential(torch.nn.Linear(24, 40), torch.nn.Tanh(), torch.nn.Linear(40, 9)).to(device, dtype)


@gpu
def test_optimizer_against_torch():
    """Five steps of torch's own AdamW on the same gradients, two groups of different options, clipped: 32-bit states, 32-bit parameters."""
    ours, theirs = model(torch.float32), model(torch.float32)
    groups = lambda net: [dict(params=net[0].parameters(), weight_decay=0.3), dict(params=net[2].parameters(), lr=2e-3, betas=(0.8, 0.95))]
    a = AdamW(groups(ours), lr=1e-2, max_norm=0.7)
    b = torch.optim.AdamW(groups(theirs), lr=1e-2)
    for k in range(5):
        torch.manual_seed(k)
        x = torch.randn(16, 24, device=DEV)
        for net, optimizer in ((ours, a), (theirs, b)):
            optimizer.zero_grad()
            net(x).square().sum().backward()
            if net is theirs:
                norm = torch.nn.utils.clip_grad_norm_(net.parameters(), 0.7)
            optimizer.step()
        assert float(a.grad_norm) == pytest.approx(float(norm), rel=1e-5)
        # both are off by some 40 u of a step of about lr, and each step's gradients by what the steps before have left of that
        for p, q in zip(ours.parameters(), theirs.parameters()):
            assert torch.allclose(p, q, rtol=1e-4, atol=1e-5), k


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_goes_on_from_a_saved_state(bits, dtype):
    def train(net, optimizer, steps):
        for k in steps:
            torch.manual_seed(k)
            optimizer.zero_grad()
            net(torch.randn(16, 24, device=DEV, dtype=dtype)).float().square().mean().backward()
            optimizer.step()

    net = model(dtype)
    optimizer = AdamW(net.parameters(), lr=1e-2, state_bits=bits, max_norm=1.0)
    train(net, optimizer, range(3))
    saved = copy.deepcopy(optimizer.state_dict()), copy.deepcopy(net.state_dict())
    train(net, optimizer, range(3, 6))
    other = model(dtype)
    other.load_state_dict(saved[1])
    again = AdamW(other.parameters(), lr=5.0, state_bits=bits, max_norm=1.0)
    again.load_state_dict(saved[0])
    assert len({id(s["step"]) for s in again.state.values()}) == 1   # one call for all of them
    for s in again.state.values():
        assert s["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn)
    train(other, again, range(3, 6))
    for p, q in zip(net.parameters(), other.parameters()):
        assert torch.equal(p, q)
    if bits == 8:   # two bytes a parameter, and the exponents
        s = optimizer.state[next(net.parameters())]
        assert s["exp_avg"].element_size() == s["exp_avg_sq"].element_size() == 1 and s["exp_avg_exponents"].numel() == (24 * 40 + 255) // 256


def test_saved_states_that_do_not_fit():
    w = torch.nn.Parameter(torch.randn(24, 40))
    optimizer = AdamW([w], state_bits=8)
    small = lambda *shape: torch.zeros(*shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
    numbers = dict(step=torch.ones(1, dtype=torch.int64), seed=torch.zeros(1, dtype=torch.int64), exp_avg_exponents=torch.zeros(4, dtype=torch.int8), exp_avg_sq_exponents=torch.zeros(4, dtype=torch.int8))
    saved = lambda m, v: dict(optimizer.state_dict(), state={0: dict(numbers, exp_avg=m, exp_avg_sq=v)})
    optimizer.load_state_dict(saved(small(24, 40), small(24, 40)))
    assert optimizer.state[w]["exp_avg"].dtype == torch.float8_e4m3fn
    for m, v in ((small(40, 24).T, small(24, 40)), (small(24, 40), small(40, 24).T), (small(40, 24), small(40, 24))):
        with pytest.raises(ValueError):
            optimizer.load_state_dict(saved(m, v))
    with pytest.raises(ValueError):
        optimizer.load_state_dict(torch.optim.AdamW([torch.nn.Parameter(torch.randn(24, 40))]).state_dict())
    one = torch.nn.Parameter(torch.randn(1, 40).T)   # an axis of one element says nothing about the order
    AdamW([one], state_bits=8).load_state_dict(saved(small(40, 1), small(40, 1)))


@gpu
def test_exponents_that_share_memory_are_refused():
    params = [torch.zeros(512, device=DEV) for _ in range(2)]
    state = lambda: [torch.zeros(512, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    e = lambda: [torch.zeros(2, dtype=torch.int8, device=DEV) for _ in range(2)]
    one, step, seed = e(), torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    for em, ev in (([one[0], one[0]], e()), (one, [one[1], one[0]])):
        with pytest.raises(ValueError, match="share memory"):
            ops.adamw_step(params, [torch.ones_like(p) for p in params], state(), state(), step, lr=1e-3, seed=seed, exp_avg_exponents=em, exp_avg_sq_exponents=ev)
    assert int(step) == 0


@gpu
def test_optimizer_with_parameters_that_join_later_and_several_types():
    net = torch.nn.ModuleList([torch.nn.Linear(8, 8, device=DEV), torch.nn.Linear(8, 8, device=DEV, dtype=torch.bfloat16), torch.nn.Linear(8, 8, device=DEV)])
    optimizer = AdamW(net.parameters(), lr=1e-2, max_norm=1.0)
    for k in range(3):
        optimizer.zero_grad(set_to_none=True)
        net[0](torch.randn(4, 8, device=DEV)).square().sum().backward()
        net[1](torch.randn(4, 8, device=DEV, dtype=torch.bfloat16)).float().square().sum().backward()
        if k == 2:
            net[2](torch.randn(4, 8, device=DEV)).square().sum().backward()
        grads = [p.grad for p in net.parameters() if p.grad is not None]
        exact = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        optimizer.step()
        assert float(optimizer.grad_norm) == pytest.approx(exact, rel=1e-6)
    steps = [int(optimizer.state[p]["step"]) for p in net.parameters()]
    assert steps == [3, 3, 3, 3, 1, 1]
    version = net[0].weight._version
    optimizer.step()
    assert net[0].weight._version > version


@gpu
def test_a_step_that_begins_inside_a_capture_is_refused():
    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    p.grad = torch.ones(8, device=DEV)
    optimizer = AdamW([p])
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before one is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            optimizer.step()
    optimizer.step()
    assert int(optimizer.state[p]["step"]) == 1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_second_moments_below_the_normal_numbers(dtype, bits):
    """Squares that begin around 2^-126 and below, alone in their 256 and beside larger ones, and fade until they are zero: states and parameters are the formula's, whose numbers of 32 bits they are formed from."""
    n, b, eps, lr = 8 * 256, 0.5, 1e-30, 3e-3
    grad = torch.exp2(-torch.arange(8.0) * 2).repeat_interleave(256)   # 1 .. 2^-14, by 256
    grad[:256:2] = 2.0 ** -12   # sizes of many orders side by side
    grad[1:256:64] = 2.0 ** -14
    grad[::7] = 0
    grad[3::5] *= -1
    grad, nothing = grad.to(dtype).to(DEV), torch.zeros(n, dtype=dtype, device=DEV)
    p, = tensors([(n,)], dtype, 1, DEV)
    (m,), (v,), em, ev = empty_states([(n,)], bits)
    step, one = counter(), torch.ones(1, device=DEV)
    scale = torch.tensor(1e-18) / (torch.ones(()) + 1e-6)   # of the gradients, by their clipping: fp16 has none of such sizes
    for t in range(1, 45):
        g = (grad if t in (1, 2, 40) else nothing).cpu().float() * scale
        p0 = p.cpu().double()
        if bits == 8:
            m0, r0 = values(m, em[0]).float(), values(v, ev[0]).float()
            v0 = r0 * r0
        else:
            m0, v0 = m.cpu(), v.cpu()
        m1, v1 = b * m0 + b * g, b * v0 + b * (g * g)
        ops.adamw_step([p], [grad if t in (1, 2, 40) else nothing], [m], [v], step, lr=lr, betas=(b, b), eps=eps, weight_decay=0.0, max_norm=1e-18, norm=one, seed=seed_of() if bits == 8 else None,
                       exp_avg_exponents=em, exp_avg_sq_exponents=ev)
        root = v1.double().sqrt()
        if bits == 8:
            check_chance(m, em[0], m1.double(), False)
            check_chance(v, ev[0], root, True)
        else:
            assert torch.equal(m.cpu(), m1) and torch.equal(v.cpu(), v1), t
        change = lr / (1 - b ** t) * m1.double() / (root / math.sqrt(1 - b ** t) + eps)
        slack = 40 * U * (p0.abs() + change.abs())
        want = p0 - change
        kind = {torch.float32: 0.0}.get(dtype, torch.finfo(dtype).eps / (2 if bits == 32 else 1))
        most = slack + kind * (want.abs() + slack).clamp(min=torch.finfo(dtype).tiny)
        # (where v has faded to zero and m has not, a step is m / eps by the formula: in fp16 a parameter passes 65504 at last, and is infinite from there on)
        far = want.abs() > torch.finfo(dtype).max
        close(p.cpu()[~far], want[~far], most[~far], t)
        assert torch.equal(p.cpu()[far].double(), torch.copysign(torch.tensor(math.inf, dtype=torch.float64), want[far]))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_elements_without_gradients_and_an_eps_of_zero(bits):
    """Parameters of 16 bits that never had a gradient stay where they are, decay aside, whatever eps is."""
    p, = tensors([(600,)], torch.bfloat16, 1, DEV)
    g = torch.zeros_like(p)
    g[7] = 0.25
    before = p.clone()
    m, v, em, ev = empty_states([(600,)], bits)
    for _ in range(2):
        ops.adamw_step([p], [g], m, v, counter(), lr=1e-2, eps=0.0, weight_decay=0.0, seed=seed_of(), exp_avg_exponents=em, exp_avg_sq_exponents=ev)
    there = torch.arange(600, device=DEV) == 7
    assert torch.equal(p[~there], before[~there]) and p.isfinite().all() and p[7] != before[7]


@gpu
def test_parameters_that_pause():
    """Parameters without a gradient in some steps, which begin together: their counts and what they become are those of torch's AdamW, which counts for each."""
    nets = [torch.nn.ModuleList(torch.nn.Linear(16, 16) for _ in range(4)) for _ in range(2)]
    nets[1].load_state_dict(nets[0].state_dict())
    ours, theirs = (net.to(DEV) for net in nets)
    a, b = AdamW(ours.parameters(), lr=1e-2, betas=(0.9, 0.99)), torch.optim.AdamW(theirs.parameters(), lr=1e-2, betas=(0.9, 0.99))
    which = [(0, 1, 2, 3)] + [(0, 1)] * 4 + [(0, 2), (0, 1, 2, 3), (3,), (), (0, 1, 2, 3), (2, 3)]
    for k, used in enumerate(which):
        for net, optimizer in ((ours, a), (theirs, b)):
            torch.manual_seed(k)
            optimizer.zero_grad(set_to_none=True)
            for i in used:
                net[i](torch.randn(8, 16, device=DEV)).square().sum().backward()
            optimizer.step()
        for i, (p, q) in enumerate(zip(ours.parameters(), theirs.parameters())):
            assert int(a.state[p]["step"]) == int(b.state[q]["step"]), (k, i)
            assert torch.allclose(p, q, rtol=1e-4, atol=1e-5), (k, i)   # as in test_optimizer_against_torch
    assert len({int(s["seed"]) for s in a.state.values()}) == len({id(s["step"]) for s in a.state.values()}) == 4
    again = AdamW(ours.parameters())
    again.load_state_dict(copy.deepcopy(a.state_dict()))
    assert [int(again.state[p]["step"]) for p in ours.parameters()] == [int(a.state[p]["step"]) for p in ours.parameters()]


@gpu
def test_a_pause_that_begins_inside_a_capture_is_refused():
    params = [torch.nn.Parameter(torch.ones(8, device=DEV)) for _ in range(2)]
    optimizer = AdamW(params, lr=1e-2)
    for p in params:
        p.grad = torch.ones(8, device=DEV)
    optimizer.step()
    params[1].grad = None
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="before one is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            optimizer.step()
    assert [int(optimizer.state[p]["step"]) for p in params] == [1, 1]
    optimizer.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        optimizer.step()
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert [int(optimizer.state[p]["step"]) for p in params] == [3 + k, 1]


def test_copies_and_pickles_keep_the_clipping():
    w = torch.nn.Parameter(torch.zeros(3))
    optimizer = AdamW([w], max_norm=0.5, lr=1e-2)
    optimizer.grad_norm = torch.ones(())
    stored = io.BytesIO()
    torch.save(optimizer, stored)
    stored.seek(0)
    for again in (copy.deepcopy(optimizer), pickle.loads(pickle.dumps(optimizer)), torch.load(stored, weights_only=False)):
        assert again.max_norm == 0.5 and again.grad_norm is None and again.param_groups[0]["lr"] == 1e-2
        assert again.step() is None   # (no gradients)


def test_saved_states_bring_their_clipping():
    make = lambda **more: AdamW([torch.nn.Parameter(torch.zeros(3))], **more)
    for max_norm in (0.5, None):
        other = make(max_norm=2.0)
        other.load_state_dict(make(max_norm=max_norm).state_dict())
        assert other.max_norm == max_norm
    before = {k: v for k, v in make().state_dict().items() if k in ("state", "param_groups")}   # (as they were saved without it)
    other = make(max_norm=2.0)
    other.load_state_dict(before)
    assert other.max_norm == 2.0


def test_a_step_without_gradients_leaves_no_norm():
    optimizer = AdamW([torch.nn.Parameter(torch.zeros(3))], max_norm=1.0)
    optimizer.grad_norm = torch.ones(())   # (of the step before)
    optimizer.step()
    assert optimizer.grad_norm is None


@pytest.mark.parametrize("seed", [1.5, "1", 2 ** 64, -2 ** 63 - 1])
def test_seeds_that_are_refused(seed):
    with pytest.raises(ValueError, match="seed"):
        AdamW([torch.nn.Parameter(torch.zeros(3))], seed=seed)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_replicas_with_one_seed_stay_together(bits):
    """Processes that draw other numbers for their data round alike if their optimizers have one seed, which takes nothing from anyone's generator; sets of parameters that begin apart have numbers of their own."""
    def run(seed, generator):
        net = model(torch.bfloat16)
        optimizer = AdamW(net.parameters(), lr=1e-3, state_bits=bits, seed=seed)
        torch.manual_seed(generator)
        state = torch.get_rng_state()
        for k in range(3):
            for i, p in enumerate(net.parameters()):
                p.grad = None if k == 0 and i == 2 else torch.full_like(p, 0.1 * (k + 1)).mul_(torch.arange(p.numel(), device=DEV).view(p.shape) % 7 - 3)
            optimizer.step()
        assert torch.equal(state, torch.get_rng_state()) == (seed is not None)
        return net, optimizer

    for seed in (0, 2 ** 64 - 1):
        (a, first), (b, _) = run(seed, 1), run(seed, 2)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
        assert len({int(s["seed"]) for s in first.state.values()}) >= 2
    for other in (run(1, 1)[0], run(None, 1)[0]):
        assert not all(torch.equal(p, q) for p, q in zip(a.parameters(), other.parameters()))
    # one seed in a group does not make sets of parameters one: each has its count behind a saved state too
    again = AdamW(a.parameters(), state_bits=bits)
    again.load_state_dict(copy.deepcopy(first.state_dict()))
    assert [int(again.state[p]["step"]) for p in a.parameters()] == [3, 3, 2, 3] and again.param_groups[0]["seed"] == 2 ** 64 - 1


@gpu
def test_exponents_that_are_written_say_so():
    (m,), (v,), em, ev = empty_states([(300,)], 8)
    p, g = tensors([(300,), (300,)], torch.bfloat16, 1, DEV)
    written = (p, m, v, *em, *ev)
    before = [t._version for t in written]
    ops.adamw_step([p], [g], [m], [v], counter(), lr=1e-3, seed=seed_of(), exp_avg_exponents=em, exp_avg_sq_exponents=ev)
    assert all(t._version > n for t, n in zip(written, before))


@gpu
def test_what_is_read_shares_no_memory_with_what_is_written():
    flat = torch.zeros(4096, device=DEV)
    p, g, m, v = (flat[1024 * i:1024 * i + 700] for i in range(4))
    good = dict(params=[p], grads=[g], exp_avgs=[m], exp_avg_sqs=[v], step=counter(), lr=1e-3)
    ops.adamw_step(**good)   # (parts of one buffer)
    number = lambda t, i, dtype: t[i:i + (8 if dtype == torch.int64 else 4) // t.element_size()].view(dtype)
    for change in (dict(grads=[p]), dict(grads=[m]), dict(grads=[flat[-924:-224]]), dict(lr=number(p, 0, torch.float32)), dict(step=number(v, 10, torch.int64)),
                   dict(seed=number(m, 698, torch.int64)), dict(max_norm=1.0, norm=number(p, 699, torch.float32))):
        with pytest.raises(ValueError, match="share"):
            ops.adamw_step(**(good | change))
    both = counter()
    with pytest.raises(ValueError, match="share"):
        ops.adamw_step(**(good | dict(step=both, seed=both)))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_of_a_count_that_change_their_type(bits):
    """Parameters that began together and are of two types later, as their module or a saved state has it: two calls, of which each counts once."""
    def step(net, optimizer):
        for p in net.parameters():
            p.grad = torch.ones_like(p)
        optimizer.step()

    make = lambda: torch.nn.ModuleList(torch.nn.Linear(16, 16, device=DEV) for _ in range(2))
    net = make()
    optimizer = AdamW(net.parameters(), state_bits=bits)
    step(net, optimizer)
    saved = copy.deepcopy(optimizer.state_dict())
    net[1].bfloat16()
    other = make()
    other[1].bfloat16()
    again = AdamW(other.parameters(), state_bits=bits)
    again.load_state_dict(saved)
    for n, o in ((net, optimizer), (other, again)):
        for k in range(2):
            step(n, o)
            assert [int(o.state[p]["step"]) for p in n.parameters()] == [2 + k] * 4


def test_seeds_of_other_kinds_of_whole_numbers():
    import numpy as np

    for seed, number in ((np.int64(-5), -5), (np.uint64(2 ** 64 - 1), 2 ** 64 - 1), (True, 1)):
        kept = AdamW([torch.nn.Parameter(torch.zeros(3))], seed=seed).param_groups[0]["seed"]
        assert type(kept) is int and kept == number
    with pytest.raises(ValueError, match="seed"):
        AdamW([torch.nn.Parameter(torch.zeros(3))], seed=torch.tensor(3))
