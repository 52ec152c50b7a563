"""Gated blocks, norms behind blocks and the scales of their branches inside `CastleLM`, their modules, and a training step of all of it with `AdamW`.

Tolerances.  In float32 the native model and the PyTorch formulation differ by roundings of 2^-24 through some ten operators a layer with sums of up to a few hundred products: 1e-4 of the largest value bounds
them with room (2e-3 for gradients, which pass through softmax and norms of small rows).  Steps on caches against whole sequences: the same operators, 2e-3 as for the models without these blocks."""
import copy

import pytest
import torch
import torch.nn.functional as F

from lookahead_keys_attention_amd import AdamW, CastleLM, GatedFeedForward, ResidualBranch, ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
KINDS = [dict(gated=True), dict(post_norm=True), dict(gated=True, post_norm=True, residual_scale=0.3), dict(gated=True, residual_scale=0.5, activation="gelu")]


def models(kind, dtype=torch.float32, **more):
    """A native model and the same one in the PyTorch formulation."""
    options = dict(num_tokens=96, dim=64, depth=2, heads=2, dim_head=32) | kind | more
    torch.manual_seed(0)
    native = CastleLM(**options, use_triton=True)
    for p in native.parameters():   # (norms of ones and scales of one number would hide a mix-up)
        if p.dim() == 1 and p.requires_grad:
            p.data.mul_(1 + 0.2 * torch.randn_like(p))
    dense = CastleLM(**options, use_triton=False)
    dense.load_state_dict(native.state_dict())
    return native.to(DEV, dtype), dense.to(DEV, dtype)


def near(a, b, tol, what):
    a, b = a.detach().double(), b.detach().double()
    off = float((a - b).abs().max() / b.abs().max())
    assert off <= tol, (what, off)


# ---- without a GPU --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_modules_are_the_formula(activation):
    torch.manual_seed(1)
    block = GatedFeedForward(24, 40, activation).double()
    x = torch.randn(3, 5, 24, dtype=torch.float64)
    u = x @ block.to_hidden.weight.T
    g, v = u[..., :40], u[..., 40:]
    act = g * torch.sigmoid(g) if activation == "silu" else g * 0.5 * torch.erfc(-g * 0.5 ** 0.5)
    assert torch.allclose(block(x), (act * v) @ block.to_out.weight.T)
    branch, norm = ResidualBranch(24, True, 0.3).double(), torch.nn.RMSNorm(24).double()
    r = torch.randn_like(x)
    y, h = branch(x, r, norm)
    want = r + torch.tensor(0.3).double() * F.rms_norm(x, (24,))   # (the scale began as a 32-bit number)
    assert torch.allclose(y, want) and torch.allclose(h, F.rms_norm(want, (24,)))
    assert GatedFeedForward(96).to_out.weight.shape == (96, 256)
    with pytest.raises(ValueError):
        GatedFeedForward(24, 40, "relu")


@pytest.mark.parametrize("kind", KINDS)
def test_models_on_the_cpu(kind):
    torch.manual_seed(2)
    lm = CastleLM(num_tokens=50, dim=32, depth=2, heads=2, dim_head=16, use_triton=False, **kind)
    ids = torch.randint(0, 50, (2, 9))
    loss = lm(ids, return_loss=True)
    loss.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in lm.parameters() if p.requires_grad)
    with torch.no_grad():
        whole, cache = lm(ids, return_next_cache=True)
        step, _ = lm(ids[:, :1], cache=cache, return_next_cache=True)
        longer = lm(torch.cat((ids, ids[:, :1]), 1))
    assert torch.allclose(longer[:, -1:], step, atol=1e-4)
    again = CastleLM(num_tokens=50, dim=32, depth=2, heads=2, dim_head=16, use_triton=False, **kind)
    again.load_state_dict(lm.state_dict())
    assert torch.equal(again(ids), lm(ids))
    assert lm.sample(ids, 12, temperature=0).shape == (2, 3)


def test_options_that_are_refused():
    with pytest.raises(ValueError):
        CastleLM(num_tokens=8, dim=32, depth=1, use_triton=False, prenorm=False, post_norm=True)
    with pytest.raises(ValueError):
        CastleLM(num_tokens=8, dim=32, depth=1, use_triton=False, gated=True, activation="relu")


def test_models_of_before_keep_their_parameters():
    names = set(CastleLM(num_tokens=8, dim=32, depth=1, use_triton=False).state_dict())
    assert not any("branch" in n or "next_norm" in n or "first_norm" in n for n in names) and "layers.0.1.3.weight" in names


# ---- on a GPU -------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_native_models_against_the_formulation(kind):
    native, dense = models(kind)
    ids = torch.randint(0, 96, (3, 41), device=DEV)
    with torch.no_grad():
        near(native(ids), dense(ids), 1e-4, "logits")
    losses = [m(ids, return_loss=True) for m in (native, dense)]
    near(*losses, 1e-4, "loss")
    for loss in losses:
        loss.backward()
    for (name, p), q in zip(native.named_parameters(), dense.parameters()):
        if p.requires_grad:
            near(p.grad, q.grad, 2e-3, name)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cached_steps_and_graphs(kind, dtype):
    native, _ = models(kind, dtype)
    ids = torch.randint(0, 96, (4, 30), device=DEV)
    tol = 2e-3 if dtype == torch.float32 else 6e-2   # (16-bit roundings of other places through two layers)
    with torch.no_grad():
        whole = native(ids)
        _, cache = native(ids[:, :20], return_next_cache=True)
        for i in range(20, 30):
            step, cache = native(ids[:, i:i + 1], cache=cache, return_next_cache=True)
            near(step[:, 0].float(), whole[:, i].float(), tol, i)
    steps = native.sample(ids[:, :12], 40, temperature=0, graph=False)
    replayed = native.sample(ids[:, :12], 40, temperature=0, graph=True)
    assert torch.equal(native.sample(ids[:, :12], 40, temperature=0, graph=True), replayed)
    if dtype == torch.float32:
        assert torch.equal(steps, replayed)
    # (in 16 bits two classes may be nearer to each other than the roundings of the attention's splits, which differ between the two: each pick is the largest logit of the whole pass within them)
    for picked in (steps, replayed):
        with torch.no_grad():
            logits = native(torch.cat((ids[:, :12], picked), 1))[:, 11:-1].float()
        behind = logits.amax(-1) - logits.gather(-1, picked[..., None])[..., 0]
        assert float(behind.max()) <= tol * float(logits.abs().max())


@gpu
def test_what_goes_through_the_kernels(monkeypatch):
    """The native model's blocks call the operators, with hooks on a module that would be passed by they call the modules."""
    native, _ = models(dict(gated=True, post_norm=True, residual_scale=0.3), torch.bfloat16)
    seen = []
    for name in ("gated_feed_forward", "residual_norm"):
        monkeypatch.setattr(ops, name, lambda *a, _f=getattr(ops, name), _n=name, **k: (seen.append(_n), _f(*a, **k))[1])
    ids = torch.randint(0, 96, (2, 17), device=DEV)
    with torch.no_grad():
        want = native(ids)
        assert seen.count("gated_feed_forward") == 2 and seen.count("residual_norm") == 4
        seen.clear()
        calls = []
        hooks = [native.next_norms[0].register_forward_hook(lambda *a: calls.append(0)), native.layers[0][1][0].to_out.register_forward_hook(lambda *a: calls.append(1))]
        got = native(ids)
        assert sorted(calls) == [0, 1] and seen.count("gated_feed_forward") == 1 and seen.count("residual_norm") == 3
        near(got.float(), want.float(), 6e-2, "with hooks")
        for hook in hooks:
            hook.remove()
        seen.clear()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            native.float()(ids)
        assert not seen


@gpu
@pytest.mark.parametrize("next_norm", [torch.nn.RMSNorm(16, elementwise_affine=False), torch.nn.RMSNorm((3, 16)), torch.nn.RMSNorm(16)])
@pytest.mark.parametrize("own", [torch.nn.RMSNorm(16, elementwise_affine=False), torch.nn.RMSNorm((3, 16)), None])
def test_branches_with_other_norms(next_norm, own):
    """Norms without weights or over more than a row: the formulation."""
    branch = ResidualBranch(16, False, 0.3, use_triton=True)
    branch.norm = own
    branch, next_norm = branch.to(DEV), copy.deepcopy(next_norm).to(DEV)
    x, r = torch.randn(2, 3, 16, device=DEV), torch.randn(2, 3, 16, device=DEV)
    y, h = branch(x, r, next_norm)
    want = r + 0.3 * (x if own is None else own.to(DEV)(x))
    near(y, want, 1e-6, "sum")
    near(h, next_norm(want), 1e-5, "norm")


@gpu
def test_loss_over_a_large_vocabulary_and_dropout():
    kind = dict(gated=True, post_norm=True, residual_scale=0.4, num_tokens=20000, embedding_scale=8.0)
    native, dense = models(kind, torch.bfloat16)
    ids = torch.randint(0, 20000, (4, 300), device=DEV)
    losses = [m(ids, return_loss=True) for m in (native, dense)]
    near(*losses, 1e-2, "loss")
    for loss in losses:
        loss.backward()
    g, w = native.to_logits.weight.grad.float(), dense.to_logits.weight.grad.float()
    assert float((g - w).norm() / w.norm()) < 5e-2
    native.dropout = 0.2
    native.train()
    with torch.no_grad():
        torch.manual_seed(5)
        a, b = native(ids), native(ids)
        torch.manual_seed(5)
        assert not torch.equal(a, b) and torch.equal(a, native(ids))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_training_step_of_all_of_it(bits):
    """Embedding, attention, gated blocks, norms and scales, loss, clipping and AdamW of a bf16 model: gradients against the formulation's, the update against the formula from those gradients, the same in a graph."""
    kind = dict(gated=True, post_norm=True, residual_scale=0.3)
    native, dense = models(kind, torch.bfloat16)
    native.train()
    ids = torch.randint(0, 96, (4, 65), device=DEV)
    params = [p for p in native.parameters() if p.requires_grad]
    optimizer = AdamW(params, lr=1e-3, weight_decay=0.1, max_norm=0.5, state_bits=bits, stochastic_rounding=False)
    before = [p.detach().clone() for p in params]

    def step():
        optimizer.zero_grad(set_to_none=False)
        loss = native(ids, return_loss=True)
        loss.backward()
        optimizer.step()
        return loss.detach()

    step()
    dense(ids, return_loss=True).backward()
    theirs = [p.grad for p in dense.parameters() if p.requires_grad]
    for p, q in zip(params, theirs):
        assert float((p.grad.float() - q.float()).norm() / q.float().norm()) < 0.1   # 16-bit roundings of other places through two layers and back
    norm = torch.cat([p.grad.flatten().double() for p in params]).norm()
    assert abs(float(optimizer.grad_norm) - float(norm)) <= 1e-6 * float(norm)
    clip = min(1.0, 0.5 / (float(norm) + 1e-6))
    for p, old in zip(params, before):
        g = p.grad.double() * clip
        want = old.double() * (1 - 1e-4) - 1e-3 * g / (g.abs() + 1e-8)   # (of the first step)
        # half a step of the type, with 8-bit states a whole one: those round parameters by chance too
        most = want.abs().clamp(min=2.0 ** -126) * (2.0 ** -8 if bits == 32 else 2.0 ** -7) + 1e-3 * 1e-5 + 1e-8
        assert ((p.detach().double() - want).abs() <= most * 1.01).all()
    # two steps outside, two replayed
    state = copy.deepcopy(optimizer.state_dict()), [p.detach().clone() for p in params]
    eager = [(step(), [p.detach().clone() for p in params]) for _ in range(2)]
    optimizer.load_state_dict(state[0])
    with torch.no_grad():
        for p, old in zip(params, state[1]):
            p.copy_(old)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        for p in params:
            p.grad.zero_()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        optimizer.zero_grad(set_to_none=False)
        loss = native(ids, return_loss=True)
        for p, g in zip(params, torch.autograd.grad(loss, params)):
            p.grad.copy_(g)
        optimizer.step()
    # The library's loss over (batch, classes, positions) adds its partial sums, one for each of the 4 sequences, to a bf16 number in any order: after each of 4 additions and the division
    # half a step, so two orders are up to 2 (4 + 1) 2^-9 of it apart.  Nothing else depends on that number.
    for want, after in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(loss.detach()) - float(want)) <= 10 * 2.0 ** -9 * float(want)
        assert all(torch.equal(p, q) for p, q in zip(params, after))


@gpu
@pytest.mark.parametrize("kind", [dict(gated=True), dict(gated=True, post_norm=True)])
def test_a_kept_decoder_and_another_gate(kind):
    """What a graph of a token step has recorded and a module may change: tokens are those of the modules as they are."""
    native, _ = models(kind)
    prompt = torch.randint(0, 96, (4, 12), device=DEV)
    first = native.sample(prompt, 40, temperature=0, graph=True)
    for _, feed_forward in native.layers:
        feed_forward[-1].activation = "gelu"
        feed_forward[-1].to_out.weight.data.mul_(4)   # (so that the gate decides tokens)
    want = native.sample(prompt, 40, temperature=0, graph=False)
    kept = native._kept_decoder
    assert torch.equal(native.sample(prompt, 40, temperature=0, graph=True), want)
    assert native._kept_decoder is not kept and not torch.equal(first, want)
    kept = native._kept_decoder
    native.sample(prompt, 40, temperature=0, graph=True)
    assert native._kept_decoder is kept
    native.layers[0][1][-1].use_triton = False
    native.sample(prompt, 40, temperature=0, graph=True)
    assert native._kept_decoder is not kept
    if kind.get("post_norm"):
        kept = native._kept_decoder
        native.next_norms[0].eps = 1.0
        assert torch.equal(native.sample(prompt, 40, temperature=0, graph=True), native.sample(prompt, 40, temperature=0, graph=False))
        assert native._kept_decoder is not kept


@gpu
def test_branches_whose_sums_are_broadcast():
    """Shapes that only add up by broadcasting: the formulation."""
    branch, norm = ResidualBranch(24, True, 0.3, use_triton=True).to(DEV), torch.nn.RMSNorm(24).to(DEV)
    x, r = torch.randn(3, 5, 24, device=DEV), torch.randn(1, 5, 24, device=DEV)
    for a, b in ((x, r), (r, x), (x, r[0, 0])):
        y, h = branch(a, b, norm)
        want = b + 0.3 * F.rms_norm(a, (24,))
        near(y, want, 1e-6, "sum")
        near(h, F.rms_norm(want, (24,)), 1e-5, "norm")
    branch.scale = torch.nn.Parameter(torch.full((1,), 0.5, device=DEV))   # (one number for all columns)
    near(branch(x, x, norm)[0], x + 0.5 * F.rms_norm(x, (24,)), 1e-6, "sum")


@gpu
def test_hooks_on_all_modules_see_those_of_blocks_and_branches():
    block, branch, norm = GatedFeedForward(24, 40, use_triton=True).to(DEV), ResidualBranch(24, True, 0.3, use_triton=True).to(DEV), torch.nn.RMSNorm(24).to(DEV)
    x, seen = torch.randn(3, 5, 24, device=DEV), []
    want = branch(block(x), x, norm)
    hook = torch.nn.modules.module.register_module_forward_hook(lambda module, *_: seen.append(module))
    try:
        got = branch(block(x), x, norm)
    finally:
        hook.remove()
    assert {id(m) for m in seen} == {id(m) for m in (block, block.to_hidden, block.to_out, branch, branch.norm, norm)}
    for a, b in zip(got, want):
        near(a, b, 1e-4, "with hooks")
