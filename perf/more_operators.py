"""The operators of a gated transformer block and of its training step, as they are timed: the gated feed-forward block, the
norms around a block with its gate and residual scale, the AdamW step over many tensors with clipped gradients.

`run` computes them in elementary torch operations in 32 bits (`own` false) or through this package's entry points:
  ops.gated_feed_forward(x, weight_in, weight_out, activation)    (act(x G^T) * (x U^T)) weight_out^T, weight_in = [G; U] (2 F, D), weight_out (D, F)
  ops.residual_norm(x, residual, weight, scale, gate, next_weight)
                                                                  y = residual + scale * gate * norm(x) * weight, h = norm(y) * next_weight
  ops.adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=, betas=, eps=, weight_decay=, max_norm=, seed=,
                 exp_avg_exponents=, exp_avg_sq_exponents=)       in place; -> the norm of the gradients

AdamW with states of 8 bits.  256 elements one behind the other in a tensor share a power of two 2^E, the least with which the
largest of them is at most 448, and are e4m3 numbers times that: the first moment, and the square root of the second one.
They are rounded up with the probability that keeps their mean, and so are parameters of 16 bits: to the next number below
plus as many steps as fit in (what is above it + u), u one of 65536 numbers from 0 to 1; a second moment that is not zero
stays above zero.  u comes from Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3, SC
2011): elements 8 i ... 8 i + 7 of a tensor take the eight 16-bit halves, low half first, of the four words that the key `seed`
makes of the counter (4 i + kind, step, number of the tensor), of 64, 32 and 32 bits; kind 0 is the second moment, 1
the first one, 2 the parameter, and step the number of this one, from 1.
"""
import math

import numpy as np
import torch

own = False   # true: through the package's entry points

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
DEVICE = "cuda"
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.1
NORM_EPS = torch.finfo(torch.float32).eps   # the norms' own


def _gated(name, mode, B, L, dim, hidden, dtype, activation="silu"):
    return {"name": name, "op": "gated", "mode": mode, "B": B, "L": L, "dim": dim, "hidden": hidden, "dtype": dtype, "activation": activation}


def _norms(name, mode, B, L, dim, dtype, gate="none", post=True):
    return {"name": name, "op": "norms", "mode": mode, "B": B, "L": L, "dim": dim, "dtype": dtype, "gate": gate, "post": post}


def _adamw(name, depth, dim, hidden, vocabulary, dtype, bits, clip=True):
    return {"name": name, "op": "adamw", "depth": depth, "dim": dim, "hidden": hidden, "vocabulary": vocabulary, "dtype": dtype, "bits": bits, "clip": clip}


def listed():
    return [
        # a step of fine-tuning on two short texts, the width of the headline layer, two thirds of four times that inside
        _gated("gated train 2x128", "train", 2, 128, 512, 1408, "bfloat16"),
        # a training batch of the language-model configuration
        _gated("gated train 16x1024", "train", 16, 1024, 512, 1408, "bfloat16"),
        # the width of the long-context layer configuration
        _gated("gated train 4x2048 wide", "train", 4, 2048, 2048, 5504, "bfloat16"),
        # full precision, documents of no round length, the other activation
        _gated("gated train fp32 3x1000", "train", 3, 1000, 256, 680, "float32", "gelu"),
        # one token for each of 32 served sequences, the widest model
        _gated("gated tokens 32x1", "eval", 32, 1, 2048, 5504, "bfloat16"),
        # one residual branch of the language-model configuration
        _norms("norms train 16x1024", "train", 16, 1024, 512, "bfloat16"),
        # the widest model's residual stream, a gate of each sequence
        _norms("norms train 4x16384 gate", "train", 4, 16384, 2048, "bfloat16", "sequence"),
        # one token for each of 32 served sequences
        _norms("norms tokens 32x1", "eval", 32, 1, 512, "bfloat16"),
        # a small model of bytes in full precision
        _adamw("adamw fp32 2 layers", 2, 256, 704, 256, "float32", 32),
        # the 12-layer model of the language-model configuration over subwords, 16-bit parameters
        _adamw("adamw bf16 12 layers", 12, 512, 1408, 32000, "bfloat16", 32),
        # layers of the widest model, states of 8 bits
        _adamw("adamw 8 bit 4 wide layers", 4, 2048, 5504, 32000, "bfloat16", 8),
    ]


# A drawn case costs at most about what the longest listed one of its operator does: rough rates (flop/s) to bound the draw.
_ROUGH_RATE = {"float32": 1e14, "bfloat16": 8e14, "float16": 8e14}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: max(_seconds(c) for c in listed() if c["op"] == op) for op in ("gated", "norms", "adamw")}
    while True:
        op = rng.choice(["gated", "gated", "norms", "adamw"])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32", "float16"])
        mode = rng.choice(["train", "train", "train", "eval"])
        B, L = _log_int(rng, 1, 32), _log_int(rng, 1, 8192)
        if op == "gated":
            case = _gated("", mode, B, L, 8 * _log_int(rng, 2, 256), 8 * _log_int(rng, 2, 700), dtype, rng.choice(["silu", "silu", "gelu"]))
        elif op == "norms":
            case = _norms("", mode, B, L, _log_int(rng, 16, 4096) if rng.random() < 0.3 else 8 * _log_int(rng, 2, 512), dtype,
                          rng.choice(["none", "none", "sequence", "full"]), rng.random() < 0.8)
        else:
            bits = rng.choice([32, 8])
            case = _adamw("", rng.randint(1, 8), _log_int(rng, 16, 2048), _log_int(rng, 16, 5504), _log_int(rng, 64, 32000), dtype, bits, rng.random() < 0.7)
        if _seconds(case) <= most[op] and B * L * case["dim"] < 1 << 27 and B * L * case.get("hidden", 1) < 1 << 28:
            del case["name"]
            return case


def _shapes(case):
    """The parameters of a model of gated blocks: table, norms, projections."""
    d, f = case["dim"], case["hidden"]
    layer = [(d,), (6 * d, d), (d, d), (d,), (d,), (2 * f, d), (d, f), (d,)]
    return [(case["vocabulary"], d)] + case["depth"] * layer + [(d,)]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=DEVICE).mul_(std).add_(mean)

    state = {"case": case}
    if case["op"] == "adamw":
        # one buffer for all parameters, one for their gradients and one for each state, as programs that exchange gradients in one piece keep them
        shapes = _shapes(case)
        sizes = [math.prod(s) for s in shapes]
        n = sum(sizes)
        state["sizes"] = sizes
        state["p"] = normal(n, std=0.02).to(dtype)
        # gradients whose size differs from row to row, some of them zero
        state["g"] = normal(n, std=1e-3).mul_(torch.rand(n // 1000 + 1, generator=g, device=DEVICE).mul_(8).exp_().repeat_interleave(1000)[:n] / 100).to(dtype)
        state["g"][torch.rand(n, generator=g, device=DEVICE) < 0.01] = 0
        state["step"] = torch.randint(0, 2000, (1,), generator=g, device=DEVICE)
        state["seed"] = torch.randint(-2 ** 63, 2 ** 63 - 1, (1,), generator=g, device=DEVICE)
        m, v = normal(n, std=3e-4), normal(n, std=1e-3).square_()
        if case["bits"] == 32:
            state["m"], state["v"] = m, v
        else:
            # what earlier steps have left
            blocks = [-(-k // 256) for k in sizes]
            state["m"], state["v"] = (torch.empty(n, dtype=torch.float8_e4m3fn, device=DEVICE) for _ in range(2))
            state["em"], state["ev"] = (torch.empty(sum(blocks), dtype=torch.int8, device=DEVICE) for _ in range(2))
            for code, exponents, x in ((state["m"], state["em"], m), (state["v"], state["ev"], v.sqrt_())):
                for c, e, part in zip(code.split(sizes), exponents.split(blocks), x.split(sizes)):
                    power, scaled = _scaled(part)
                    e.copy_(power)
                    c.copy_(scaled.to(torch.float8_e4m3fn))
            state["blocks"] = blocks
        return state
    train, B, L, D = case["mode"] == "train", case["B"], case["L"], case["dim"]
    if case["op"] == "gated":
        F = case["hidden"]
        state["x"] = normal(B, L, D).to(dtype).requires_grad_(train)   # rows behind a norm
        state["win"] = normal(2 * F, D, std=D ** -0.5).to(dtype).requires_grad_(train)
        state["wout"] = normal(D, F, std=F ** -0.5).to(dtype).requires_grad_(train)
    else:
        # what a block gives, against a residual stream of a few times its size
        state["x"] = normal(B, L, D, std=0.5).to(dtype).requires_grad_(train)
        state["residual"] = normal(B, L, D, std=2).to(dtype).requires_grad_(train)
        state["weight"] = normal(D, std=0.1, mean=1).to(dtype).requires_grad_(train) if case["post"] else None
        state["scale"] = normal(D, std=0.05, mean=0.3).to(dtype).requires_grad_(train)
        state["next"] = normal(D, std=0.1, mean=1).to(dtype).requires_grad_(train)
        rows = {"none": None, "sequence": 1, "full": L}[case["gate"]]
        state["gate"] = None if rows is None else torch.rand(B, rows, D, generator=g, device=DEVICE).to(dtype).requires_grad_(train)
        state["dh"] = normal(B, L, D).to(dtype) if train else None
    state["dy"] = normal(B, L, D).to(dtype) if train else None
    return state


def run(state):
    case = state["case"]
    return {"gated": _run_gated, "norms": _run_norms, "adamw": _run_adamw}[case["op"]](state, case)


# ---- this package's entry points ------------------------------------------------------------------------------
def _run_gated(state, case):
    if not own:
        return _plain_gated(state, case)
    from lookahead_keys_attention_amd import ops

    x, win, wout = state["x"], state["win"], state["wout"]
    y = ops.gated_feed_forward(x, win, wout, activation=case["activation"])
    if case["mode"] == "eval":
        return y
    dx, din, dout = torch.autograd.grad(y, (x, win, wout), state["dy"])
    return {"y": y, "dx": dx, "dweight_in": din, "dweight_out": dout}


def _norm_leaves(state):
    return {k: state[k] for k in ("x", "residual", "weight", "scale", "gate", "next") if state[k] is not None}


def _run_norms(state, case):
    if not own:
        return _plain_norms(state, case)
    from lookahead_keys_attention_amd import ops

    y, h = ops.residual_norm(state["x"], state["residual"], weight=state["weight"], scale=state["scale"], gate=state["gate"], next_weight=state["next"])
    if case["mode"] == "eval":
        return {"y": y, "h": h}
    leaves = _norm_leaves(state)
    grads = torch.autograd.grad((y, h), tuple(leaves.values()), (state["dy"], state["dh"]))
    return {"y": y, "h": h, **{"d" + k: t for k, t in zip(leaves, grads)}}


def _run_adamw(state, case):
    if not own:
        return _plain_adamw(state, case)
    from lookahead_keys_attention_amd import ops

    sizes, small = state["sizes"], case["bits"] == 8
    norm = ops.adamw_step(state["p"].split(sizes), state["g"].split(sizes), state["m"].split(sizes), state["v"].split(sizes), state["step"],
                          lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, max_norm=1.0 if case["clip"] else None, seed=state["seed"],
                          exp_avg_exponents=state["em"].split(state["blocks"]) if small else None,
                          exp_avg_sq_exponents=state["ev"].split(state["blocks"]) if small else None)
    return _adamw_outputs(state, norm)


def _adamw_outputs(state, norm):
    kept = {k: state[k] for k in ("p", "m", "v", "em", "ev", "step") if k in state}
    return kept if norm is None else {**kept, "norm": norm}


# ---- the plain form: 32 bits, rounded once at the end -----------------------------------------------------------
def _plain_gated(state, case):
    with torch.no_grad():
        x, win, wout = state["x"], state["win"].float(), state["wout"].float()
        dtype, rows = x.dtype, x.reshape(-1, x.shape[-1]).float()
        g, u = (rows @ win.t()).chunk(2, dim=1)
        if case["activation"] == "silu":
            s = torch.sigmoid(g)
            act, slope = g * s, s * (1 + g * (1 - s))
        else:
            s = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
            act, slope = g * s, s + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
        h = act * u
        y = (h @ wout.t()).to(dtype).view(x.shape)
        if case["mode"] == "eval":
            return y
        dy = state["dy"].reshape(rows.shape).float()
        dh = dy @ wout
        d = torch.cat((dh * u * slope, dh * act), dim=1)
        return {"y": y, "dx": (d @ win).to(dtype).view(x.shape), "dweight_in": (d.t() @ rows).to(dtype), "dweight_out": (dy.t() @ h).to(dtype)}


def _plain_norms(state, case):
    with torch.no_grad():
        x, r = state["x"].float(), state["residual"].float()
        dtype, D = state["x"].dtype, case["dim"]
        one = torch.ones((), device=DEVICE)
        w, scale, nxt = (one if state[k] is None else state[k].float() for k in ("weight", "scale", "next"))
        gate = one if state["gate"] is None else state["gate"].float()
        inv = (x.square().mean(-1, keepdim=True) + NORM_EPS).rsqrt() if case["post"] else one
        xhat = x * inv
        y = r + scale * gate * xhat * w
        inv_y = (y.square().mean(-1, keepdim=True) + NORM_EPS).rsqrt()
        yhat = y * inv_y
        out = {"y": y.to(dtype), "h": (yhat * nxt).to(dtype)}
        if case["mode"] == "eval":
            return out
        dy, dh = state["dy"].float(), state["dh"].float()
        dn = dh * nxt
        dyt = dy + inv_y * (dn - yhat * (dn * yhat).mean(-1, keepdim=True))
        dxhat = dyt * scale * gate * w
        dx = inv * (dxhat - xhat * (dxhat * xhat).mean(-1, keepdim=True)) if case["post"] else dxhat
        p = dyt * xhat
        out |= {"dx": dx.to(dtype), "dresidual": dyt.to(dtype), "dnext": (dh * yhat).sum((0, 1)).to(dtype), "dscale": (p * gate * w).sum((0, 1)).to(dtype)}
        if case["post"]:
            out["dweight"] = (p * gate * scale).sum((0, 1)).to(dtype)
        if state["gate"] is not None:
            dg = p * scale * w
            out["dgate"] = (dg.sum(1, keepdim=True) if case["gate"] == "sequence" else dg).to(dtype)
        return out


def _scaled(x):
    """Of each 256 elements of x the exponent E of their power of two, and x over it."""
    n = x.numel()
    blocks = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
    bits = blocks.abs().amax(dim=1).view(torch.int32)
    power = ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000)).clamp(-126, 120)
    return power.to(torch.int8), (blocks * _power(-power)[:, None]).view(-1)[:n]


def _power(e):
    return (e.int() + 127 << 23).view(torch.float32)


def _spread(e, n):
    return _power(e).repeat_interleave(256)[:n]


def _wide_product(m, c):
    """High and low word of the constant m times the words c, all in 64-bit integers without overflow."""
    low, high = c * (m & 0xFFFF), c * (m >> 16)
    return (high + (low >> 16)) >> 16, (low + ((high & 0xFFFF) << 16)) & 0xFFFFFFFF


def _halves(seed, step, number, n):
    """Three rows (kinds) of n random 16-bit numbers, the order of the module's docstring."""
    i = 4 * torch.arange((n + 7) // 8, device=DEVICE) + torch.arange(3, device=DEVICE)[:, None]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    a, b, c, d = i & 0xFFFFFFFF, i >> 32, (step & 0xFFFFFFFF).expand_as(i), torch.full_like(i, number)
    for _ in range(10):
        (ha, la), (hc, lc) = _wide_product(0xD2511F53, a), _wide_product(0xCD9E8D57, c)
        a, b, c, d = hc ^ b ^ key[0], lc, ha ^ d ^ key[1], la
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return torch.stack([w >> s & 0xFFFF for w in (a, b, c, d) for s in (0, 16)], dim=2).flatten(1)[:, :n].int()


def _to_e4m3(s, u, positive):
    """|s| <= 448 to e4m3 numbers, up where u says so; positive: what is not zero stays above it."""
    mag = s.abs()
    normal = ((mag.view(torch.int32) + (u << 4)) >> 20) - 960
    code = torch.where(mag < 2 ** -6, (mag * 512 + u.float() / 65536).floor().int(), normal)
    if positive:
        code = torch.where(mag > 0, code.clamp(min=1), code)
    code = torch.where(mag.isfinite(), code, 127) | torch.where(s.view(torch.int32) < 0, 128, 0)
    return code.to(torch.uint8).view(torch.float8_e4m3fn)


def _to_16_bits(p, u, dtype):
    bits = p.view(torch.int32)
    if dtype == torch.bfloat16:
        return torch.where(p.isfinite(), ((bits + u) & -65536).view(torch.float32), p).to(dtype)
    up = ((bits + (u >> 3)) & -8192).view(torch.float32)
    low = ((p.abs() * 2 ** 24 + u.float() / 65536).floor() * 2 ** -24).copysign(p)
    return torch.where(p.isfinite(), torch.where(p.abs() < 2 ** -14, low, up), p).to(dtype)


def _plain_adamw(state, case):
    with torch.no_grad():
        sizes, small, (b1, b2) = state["sizes"], case["bits"] == 8, BETAS
        grads = state["g"].split(sizes)
        norm, clip = None, torch.ones((), device=DEVICE)
        if case["clip"]:
            # squares of up to 2^128 in double: they neither overflow nor vanish
            norm = torch.stack([x.double().square().sum() for x in grads]).sum().sqrt().float()
            clip = (1.0 / (norm + 1e-6)).clamp(max=1.0)
        state["step"] += 1
        t = state["step"].double()
        rate, root = (LR / (1 - b1 ** t)).float(), (1 / (1 - b2 ** t).sqrt()).float()
        keep = torch.tensor(1 - LR * DECAY, device=DEVICE, dtype=torch.float32)
        blocks = state.get("blocks", [0] * len(sizes))
        each = zip(state["p"].split(sizes), grads, state["m"].split(sizes), state["v"].split(sizes),
                   state["em"].split(blocks) if small else blocks, state["ev"].split(blocks) if small else blocks)
        for number, (p, x, m, v, em, ev) in enumerate(each):
            n = p.numel()
            x = x.float() * clip
            if small or p.dtype != torch.float32:
                u = _halves(state["seed"], state["step"], number, n)
            m_old, v_old = (m.float() * _spread(em, n), (v.float() * _spread(ev, n)).square()) if small else (m, v)
            m_new, v_new = b1 * m_old + (1 - b1) * x, b2 * v_old + (1 - b2) * (x * x)
            r = v_new.sqrt()
            q = p.float() * keep - rate * m_new / (r * root + EPS)
            if small:
                for code, exponents, value, kind in ((v, ev, r, 0), (m, em, m_new, 1)):
                    power, s = _scaled(value)
                    exponents.copy_(power)
                    code.copy_(_to_e4m3(s, u[kind], kind == 0))
            else:
                m.copy_(m_new)
                v.copy_(v_new)
            p.copy_(q if p.dtype == torch.float32 else _to_16_bits(q, u[2], p.dtype))
        return _adamw_outputs(state, norm)


# ---- what a pass cannot do without -----------------------------------------------------------------------------
def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["op"] == "adamw":
        n = float(sum(math.prod(s) for s in _shapes(case)))
        states = 4 * (4 if case["bits"] == 32 else 1 + 1 / 256)   # two of them, read and written
        # parameters read and written, gradients read; once more for their norm, which has to be there before the first step
        return {"bytes": n * (es * (4 if case["clip"] else 3) + states), "flops": 16.0 * n}
    rows, D, train = float(case["B"]) * case["L"], case["dim"], case["mode"] == "train"
    if case["op"] == "norms":
        gates = {"none": 0.0, "sequence": float(case["B"]), "full": rows}[case["gate"]]
        # x, residual, y, h; dy, dh, x and residual again, dx, dresidual; the gate and its gradient
        return {"bytes": es * D * (rows * (10 if train else 4) + gates * (3 if train else 1)), "flops": D * rows * (34 if train else 10)}
    weights, F = 3.0 * D * case["hidden"], case["hidden"]
    # x, y, both weights; x, dy and the weights again, the gradients
    return {"bytes": es * (rows * D * (5 if train else 2) + weights * (3 if train else 1)), "flops": 6.0 * rows * D * F * (3 if train else 1)}


def _seconds(case):
    w = work(case)
    return w["bytes"] / 4e12 + (w["flops"] / _ROUGH_RATE[case["dtype"]] if case["op"] == "gated" else 0)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------
def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
    return {"gated": _exact_gated, "norms": _exact_norms, "adamw": _exact_adamw}[case["op"]](state, case)


def _exact_gated(state, case):
    """The formula in double precision; gradients by torch's own differentiation of it, a range of rows at a time."""
    x, win, wout = (state[k].detach().double() for k in ("x", "win", "wout"))
    act = torch.nn.functional.silu if case["activation"] == "silu" else torch.nn.functional.gelu
    rows, F, train = x.flatten(0, 1), case["hidden"], case["mode"] == "train"
    win.requires_grad_(train)
    wout.requires_grad_(train)
    ys, dxs = [], []
    for first in range(0, len(rows), 4096):
        part = rows[first:first + 4096].clone().requires_grad_(train)
        hidden = torch.nn.functional.linear(part, win)
        y = torch.nn.functional.linear(act(hidden[:, :F]) * hidden[:, F:], wout)
        ys.append(y.detach())
        if train:
            y.backward(state["dy"].flatten(0, 1)[first:first + 4096].double())
            dxs.append(part.grad)
    y = torch.cat(ys).view(x.shape)
    return {"y": y, "dx": torch.cat(dxs).view(x.shape), "dweight_in": win.grad, "dweight_out": wout.grad} if train else y


def _exact_norms(state, case):
    train = case["mode"] == "train"
    leaf = {k: v.detach().double().requires_grad_(train) for k, v in _norm_leaves(state).items()}
    normed = leaf["x"]
    if case["post"]:
        normed = torch.nn.functional.rms_norm(normed, (case["dim"],), leaf["weight"], NORM_EPS)
    branch = normed * leaf["scale"]
    if "gate" in leaf:
        branch = branch * leaf["gate"]
    y = leaf["residual"] + branch
    h = torch.nn.functional.rms_norm(y, (case["dim"],), leaf["next"], NORM_EPS)
    out = {"y": y.detach(), "h": h.detach()}
    if train:
        torch.autograd.backward((y, h), (state["dy"].double(), state["dh"].double()))
        out |= {"d" + k: t.grad for k, t in leaf.items()}
    return out


def _exact_adamw(state, case):
    """All tensors as one; where numbers are rounded up or down by chance, what they stand for before that."""
    sizes, (b1, b2), small = state["sizes"], BETAS, case["bits"] == 8
    g, p = state["g"].double(), state["p"].double()
    norm = torch.linalg.vector_norm(g)
    if case["clip"]:
        g = g * torch.clamp(1.0 / (norm + 1e-6), max=1.0)
    if small:
        def per_element(e):   # 2^E of every element
            return torch.cat([torch.repeat_interleave(torch.exp2(x.double()), 256)[:k] for x, k in zip(e.split(state["blocks"]), sizes)])

        m, v = state["m"].double() * per_element(state["em"]), (state["v"].double() * per_element(state["ev"])) ** 2
    else:
        m, v = state["m"].double(), state["v"].double()
    t = int(state["step"]) + 1
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g * g, v, b2)
    p = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + EPS)
    out = {"p": p, "step": None}
    if small:
        for name, x in (("m", m), ("v", torch.sqrt(v))):
            parts = []
            for part in x.split(sizes):
                k = part.numel()
                wide = torch.cat((part, part.new_zeros(-k % 256))).view(-1, 256)
                top = torch.linalg.vector_norm(wide, ord=float("inf"), dim=1)
                least = torch.ceil(torch.log2(top / 448)).clamp(-126, 120)   # the least power of two with top <= 448 times it
                parts.append((wide * torch.exp2(-least)[:, None]).flatten()[:k])
            out[name] = torch.cat(parts)
        out |= {"em": None, "ev": None}
    else:
        out |= {"m": m, "v": v}
    return {**out, "norm": norm} if case["clip"] else out
