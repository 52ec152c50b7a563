"""The language model over a large vocabulary: scaled embedding, dropout between the blocks and the loss without logits, together as training and sampling
run them.  The dense PyTorch formulation of the model (use_triton=False) in 64 bits is the reference."""
import pytest
import torch
import torch.nn.functional as F

from lookahead_keys_attention_amd import CastleLM, ops
from lookahead_keys_attention_amd import lm as LM

DEV = "cuda:0"
gpu = pytest.mark.gpu
V = 16400   # just beyond LINEAR_LOSS_MIN_VOCABULARY, no multiple of a tile


def make(native, **kw):
    torch.manual_seed(3)
    kw = {"num_tokens": V, "dim": 64, "depth": 2, "heads": 2, "dim_head": 32, **kw}
    return CastleLM(use_triton=native, **kw)


def ids(B=3, n=41, seed=0):
    return torch.randint(0, V, (B, n), generator=torch.Generator().manual_seed(seed))


# ---- without a GPU --------------------------------------------------------------------------------------------------
def test_scale_and_dropout_of_the_dense_model():
    plain, scaled = make(False).double(), make(False, embedding_scale=3.0, dropout=0.25).double()
    scaled.load_state_dict(plain.state_dict())
    x = ids()
    with torch.no_grad():
        plain.token_emb.weight.mul_(3)
    scaled.eval()
    assert torch.allclose(scaled(x), plain(x), rtol=1e-12, atol=1e-12)
    scaled.train()
    torch.manual_seed(1)
    a = scaled(x)
    assert not torch.allclose(a, plain(x))
    torch.manual_seed(1)
    assert torch.equal(scaled(x), a)
    # passes with caches drop nothing: what a sampler prefills is what it steps from
    logits, cache = scaled(x, return_next_cache=True)
    assert torch.allclose(logits, plain(x), rtol=1e-12, atol=1e-12)
    for bad in (-0.1, 1.1):
        with pytest.raises(ValueError):
            make(False, dropout=bad)
    del plain.__dict__["dropout"], plain.__dict__["embedding_scale"]   # a model that was saved whole before it had them
    assert plain(x).shape == (3, 41, V)


def test_where_the_loss_is_taken_without_logits():
    def ahead(rows, V, D, dtype=torch.bfloat16):
        return LM.linear_loss_is_ahead(rows, torch.empty(V, D, dtype=dtype, device="meta"))

    assert ahead(2048, 16384, 512) and not ahead(2048, 16383, 512) and ahead(1 << 24, 1 << 22, 512) and ahead(1, 16384, 1 << 16)
    assert not any(ahead(*bad) for bad in ((2048, (1 << 22) + 1, 512), (2048, 16384, 516), (2048, 16384, (1 << 16) + 8), (0, 16384, 512), ((1 << 24) + 1, 16384, 512)))
    # in 16 bits with gradients, wide rows go by the logits' memory
    assert ahead(2048, 32000, 520) and not ahead(2049, 32000, 520) and ahead(2049, 32000, 520, torch.float32)
    assert not ahead(1023, 16384, 64, torch.float32) and ahead(1024, 16384, 64, torch.float32)
    assert not ahead(1 << 14, 1 << 17, 1024) and ahead((1 << 14) + 1, 1 << 17, 1024)
    with torch.no_grad():
        assert ahead(2049, 32000, 520) and ahead(1, 16384, 8, torch.float32)


# ---- on a GPU -------------------------------------------------------------------------------------------------------
def train(model, x):
    model.zero_grad()
    loss = model(x, return_loss=True)
    loss.backward()
    return [loss.detach()] + [p.grad for p in model.parameters() if p.grad is not None]


@gpu
@pytest.mark.parametrize("tie", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step_equals_the_dense_model(tie, dtype, monkeypatch):
    """Loss and every gradient; with a hook the model runs module by module and forms logits, without one it does not, whatever the rule says.  bf16: the rule of the package, 2e-2 of the norm."""
    native = make(True, tie_embedding=tie, embedding_scale=8.0).to(dtype).to(DEV)
    dense = make(False, tie_embedding=tie, embedding_scale=8.0).double().to(DEV)
    dense.load_state_dict({k: v.double() for k, v in native.state_dict().items()})
    x = ids().to(DEV)
    assert native._plain(x)
    monkeypatch.setattr(LM, "linear_loss_is_ahead", lambda rows, weight: True)
    want = train(dense, x)
    tol = 1e-4 if dtype is torch.float32 else 2e-2
    for hooked in (False, True):
        handle = native.final_norm.register_forward_hook(lambda *_: None) if hooked else None
        for k, (a, b) in enumerate(zip(train(native, x), want, strict=True)):
            assert (a.double() - b).norm() <= tol * b.norm(), (hooked, k)
        if hooked:
            handle.remove()
    with torch.no_grad():   # (short sequences of 16 bits go another way without gradients: the same loss, not the same bits)
        assert (native(x, return_loss=True).double() - want[0]).abs() <= tol * want[0].abs()


@gpu
def test_wide_rows_with_and_without_logits(monkeypatch):
    """Training in bf16 on either side of the rule: the same loss and gradients within what the rounding of logits and of bf16 allows, 2e-2 of the norm."""
    model = make(True, dim=520, depth=1).bfloat16().to(DEV)
    x = ids(53, 41).to(DEV)
    assert not LM.linear_loss_is_ahead(53 * 40, model.to_logits.weight)
    want = train(model, x)
    monkeypatch.setattr(LM, "LOGITS_MAX_BYTES", 0)
    assert LM.linear_loss_is_ahead(53 * 40, model.to_logits.weight)
    for k, (a, b) in enumerate(zip(train(model, x), want, strict=True)):
        assert (a.float() - b.float()).norm() <= 2e-2 * b.float().norm(), k


@gpu
def test_no_logits_in_memory(monkeypatch):
    """The loss of 8 x 512 tokens over 131072 takes less than a quarter of the logits' memory."""
    model = CastleLM(num_tokens=131072, dim=64, depth=1, heads=2, dim_head=32).to(DEV).bfloat16()
    x = torch.randint(0, 131072, (8, 1025), device=DEV)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        loss = model(x, return_loss=True)
    assert torch.cuda.max_memory_allocated() - before < 8 * 1024 * 131072 * 2 // 4
    monkeypatch.setattr(LM, "LINEAR_LOSS_MIN_VOCABULARY", 1 << 30)
    with torch.no_grad():   # (with rounded logits: half a step of bf16 of a logit, and of the loss)
        assert (model(x, return_loss=True) - loss).abs() <= 2 * 2 ** -8 * loss.abs()


@gpu
@pytest.mark.parametrize("hooked", [False, True])
def test_dropout_in_training(hooked):
    """The masks come from the device's generator, one for each branch; the gradients are those of the same masks."""
    p = 0.25
    model = make(True, dropout=p, embedding_scale=2.0).to(DEV)
    if hooked:
        model.final_norm.register_forward_hook(lambda *_: None)
    x = ids().to(DEV)
    torch.manual_seed(7)
    got = train(model, x)
    torch.manual_seed(7)
    again = train(model, x)
    if not hooked:   # (module by module the library's loss of transposed logits is summed by atomic additions, in an order of their own)
        assert all(torch.equal(a, b) for a, b in zip(again, got))
    assert abs(train(model, x)[0] - got[0]) > 10 * abs(again[0] - got[0])
    # by hand: the dense model of 64 bits with the masks of the same numbers
    dense = make(False, embedding_scale=2.0).double().to(DEV)
    dense.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    torch.manual_seed(7)
    seeds = iter(torch.randint(-2 ** 63, 2 ** 63 - 1, (5, 2), device=DEV))

    def drop(t):
        mask = ops.dropout_add(torch.ones(t.shape, device=DEV), None, p, next(seeds))
        return t * mask.double()

    tokens, target = x[:, :-1], x[:, 1:]
    h = drop(dense.token_emb(tokens) * 2)
    for attention, feed_forward in dense.layers:
        h = h + drop(attention(h))
        h = h + drop(feed_forward(h))
    loss = F.cross_entropy(dense.to_logits(dense.final_norm(h)).transpose(1, 2), target)
    loss.backward()
    want = [loss.detach()] + [q.grad for q in dense.parameters() if q.grad is not None]
    for a, b in zip(got, want, strict=True):
        assert (a.double() - b).norm() <= 1e-4 * b.norm()
    model.eval()
    with torch.no_grad():
        a = model(x)
        assert torch.equal(a, model(x))


@gpu
def test_dropout_under_autocast():
    """The blocks' outputs have 16 bits then, what they are added to 32: the loss without dropout to within 2e-2, gradients of everything."""
    model = make(True, dropout=0.2, embedding_scale=2.0).to(DEV)
    x = ids().to(DEV)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = train(model, x)
    assert len(got) == 1 + sum(p.requires_grad for p in model.parameters()) and all(t.isfinite().all() for t in got)
    model.eval()
    with torch.no_grad():
        want = model(x, return_loss=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert (model(x, return_loss=True) - want).abs() <= 2e-2 * want


@gpu
def test_training_step_in_a_graph(monkeypatch):
    """Loss and gradients of a model, captured; each replay draws the masks that the device's generator has next, as an eager step does, and sees the tokens that are there then."""
    monkeypatch.setattr(LM, "linear_loss_is_ahead", lambda rows, weight: True)
    model = make(True, dropout=0.25, embedding_scale=2.0).bfloat16().to(DEV)
    x, leaves = ids().to(DEV), [p for p in model.parameters() if p.requires_grad]

    def step():
        loss = model(x, return_loss=True)
        return loss.detach(), *torch.autograd.grad(loss, leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    seen = []
    for k in range(3):
        x.copy_(ids(seed=k))
        torch.manual_seed(k // 2)
        want = step()
        torch.manual_seed(k // 2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        seen.append(got[1].clone())   # (a loss of 16 bits may well be the same)
    assert not any(torch.equal(seen[a], seen[b]) for a, b in ((0, 1), (0, 2), (1, 2)))


@gpu
@pytest.mark.parametrize("graph", [False, True])
def test_sampling_with_a_scaled_embedding(graph):
    """Greedy tokens of the native model, also one that is in training and has dropout, are those of the parallel pass over what it has written."""
    model = make(True, embedding_scale=4.0, dropout=0.5, num_tokens=300).to(DEV)
    prompt = torch.randint(0, 300, (2, 9), generator=torch.Generator().manual_seed(5)).to(DEV)
    new = model.sample(prompt, 25, temperature=0, graph=graph)
    model.eval()
    with torch.no_grad():
        logits = model(torch.cat((prompt, new), dim=1))
    # (a tie within rounding may go either way)
    best, took = logits[:, 8:-1].max(-1).values, logits[:, 8:-1].gather(2, new[..., None])[..., 0]
    assert (best - took <= 1e-3 * logits.abs().max()).all()


@gpu
def test_a_run_of_the_three_operators_in_a_graph():
    """Embedding, dropout, loss and their gradients, captured and replayed with other tokens and numbers."""
    torch.manual_seed(0)
    table, head = (torch.randn(3000, 64, device=DEV, requires_grad=True) for _ in range(2))
    x, seed = torch.randint(0, 3000, (4, 65), device=DEV), torch.tensor([1, 2], device=DEV)

    def step():
        h = ops.embedding(table, x[:, :-1], 8.0)
        h = ops.dropout_add(h, h, 0.1, seed)
        loss = ops.linear_cross_entropy(h, head, x[:, 1:])
        return loss.detach(), *torch.autograd.grad(loss, (table, head))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(3):
        x.copy_(torch.randint(0, 3000, (4, 65), device=DEV))
        x[0, 5:9] = -100 if k else 7
        x[0, 4:8] = x[0, 5:9].clamp(min=0)
        seed.add_(1)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) or (a.isnan() == b.isnan()).all() for a, b in zip(got, want))
        assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(got, want))
