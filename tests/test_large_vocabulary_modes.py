"""A language model's scaled embedding, dropout and loss over a large vocabulary on the passes beside plain training: a decoder that is kept between samples, sequences of one token, frozen
models, empty batches."""
import pytest
import torch

from lookahead_keys_attention_amd import CastleLM, _native, ops
from lookahead_keys_attention_amd import lm as LM

DEV = "cuda:0"
gpu = pytest.mark.gpu


def make(native=True, **kw):
    torch.manual_seed(3)
    return CastleLM(use_triton=native, **{"num_tokens": 300, "dim": 64, "depth": 2, "heads": 2, "dim_head": 32, **kw}).to(DEV)


@gpu
def test_a_kept_decoder_follows_the_scale_of_the_embedding():
    """The scale is set between two samples: the steps of the second one are those of a decoder captured anew, with the new scale."""
    model = make()
    prompt = torch.randint(0, 300, (2, 9), generator=torch.Generator().manual_seed(5)).to(DEV)

    def sample():
        return model.sample(prompt, 40, temperature=0, graph=True)

    want = {}
    for scale in (1.0, 6.0, 0.25):
        model.embedding_scale = scale
        model.release_decoder()
        want[scale] = sample()
    assert not torch.equal(want[1.0], want[6.0]) and not torch.equal(want[6.0], want[0.25])
    for scale in (6.0, 1.0, 0.25, 0.25, 1.0):
        model.embedding_scale = scale
        assert torch.equal(sample(), want[scale]), scale
        kept = model.__dict__["_kept_decoder"]
        assert torch.equal(sample(), want[scale]) and model.__dict__["_kept_decoder"] is kept   # (and the same scale again needs no other graph)


@gpu
def test_one_token_a_sequence_drops_every_branch():
    """A model in training, sequences of one token: the outputs of all blocks are dropped.  The dense model of 64 bits with the masks of the same numbers; 1e-4 of
    the norm, as for longer sequences."""
    p = 0.5
    model = make(dropout=p, embedding_scale=2.0)
    x = torch.randint(0, 300, (7, 1), generator=torch.Generator().manual_seed(6)).to(DEV)
    torch.manual_seed(9)
    with torch.no_grad():
        got = model(x)
    dense = make(False, embedding_scale=2.0).double()
    dense.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    torch.manual_seed(9)
    seeds = iter(torch.randint(-2 ** 63, 2 ** 63 - 1, (5, 2), device=DEV))
    with torch.no_grad():
        def drop(t):
            return t * ops.dropout_add(torch.ones(t.shape, device=DEV), None, p, next(seeds)).double()

        h = drop(dense.token_emb(x) * 2)
        for attention, feed_forward in dense.layers:
            h = h + drop(attention(h, return_next_cache=False))
            h = h + drop(feed_forward(h))
        want = dense.to_logits(dense.final_norm(h))
    assert (got.double() - want).norm() <= 1e-4 * want.norm()


@gpu
@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_no_tokens_at_all_still_record_a_graph(scale):
    """The embedding of an empty batch hangs on its table, whose gradient is zeros."""
    table = torch.randn(30, 16, device=DEV, requires_grad=True)
    for shape in ((0, 5), (4, 0)):
        y = _native.host().embedding(table, torch.zeros(shape, dtype=torch.long, device=DEV), scale)
        assert y.shape == (*shape, 16) and y.requires_grad
        grad, = torch.autograd.grad(y.sum(), table)
        assert grad.shape == table.shape and not grad.any()


@gpu
def test_gradient_of_few_tokens_over_a_large_vocabulary_takes_no_second_table():
    """The model's embedding of 128 tokens over 131072 rows: beside the gradient itself there is no table of partial sums in memory."""
    table = torch.randn(131072, 256, device=DEV).bfloat16().requires_grad_()
    index = torch.randint(0, 131072, (2, 64), device=DEV)
    y = _native.host().embedding(table, index)
    dy = torch.randn_like(y)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    grad, = torch.autograd.grad(y, table, dy)
    assert torch.cuda.max_memory_allocated() - before < 1.1 * grad.numel() * grad.element_size()
    want = torch.zeros(table.shape, dtype=torch.float64, device=DEV).index_add_(0, index.flatten(), dy.double().flatten(0, 1))
    assert ((grad.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()


@gpu
def test_a_model_without_gradients_takes_the_loss_of_inference(monkeypatch):
    """Frozen parameters record no graph, whether gradients are switched off or not: the rule is asked as for inference; one parameter that is not frozen, and it is asked as for training."""
    model = make(num_tokens=16400).bfloat16()
    x, asked = torch.randint(0, 16400, (3, 20), device=DEV), []
    monkeypatch.setattr(LM, "linear_loss_is_ahead", lambda rows, weight: asked.append(torch.is_grad_enabled()) or True)
    loss = model(x, return_loss=True)
    assert asked == [True] and loss.requires_grad
    model.requires_grad_(False)
    assert not model(x, return_loss=True).requires_grad and asked == [True, False]
    model.final_norm.weight.requires_grad_(True)
    assert model(x, return_loss=True).requires_grad and asked == [True, False, True]
    with torch.no_grad():
        model(x, return_loss=True)
    assert asked == [True, False, True, False]


def test_where_logits_in_memory_are_ahead():
    """Sizes on either side of each bound, in training and without gradients; logits of more than LOGITS_MAX_BYTES are never formed."""
    def ahead(rows, V, D, dtype):
        return LM.linear_loss_is_ahead(rows, torch.empty(V, D, dtype=dtype, device="meta"))

    half, full, most = torch.bfloat16, torch.float32, LM.LOGITS_MAX_BYTES
    for grad, yes, no in ((True, [(2048, 16384, 1024, half), (1024, 131072, 2048, half), (512, 16384, 4096, half), (1 << 14, 32000, 512, half), (256, 131072, 512, full),
                                  (1024, 131072, 2048, full)],
                           [(2048, 16384, 1032, half), (1025, 131072, 2048, half), (2048, 131072, 4096, half), (255, 131072, 512, full), (1023, 131072, 2048, full), (128, 131072, 2048, full)]),
                          (False, [(1, 16384, 2048, half), (1 << 14, 16384, 2048, half), (1024, 16384, 4096, half), (1, 16384, 128, full), (128, 16384, 512, full), (512, 16384, 2048, full)],
                           [(1025, 16384, 4096, half), (8192, 32000, 4096, half), (1, 16384, 136, full), (127, 16384, 512, full), (511, 131072, 2048, full)])):
        with torch.set_grad_enabled(grad):
            assert all(ahead(*case) for case in yes) and not any(ahead(*case) for case in no), grad
            for dtype in (half, full):
                rows = most // dtype.itemsize // (1 << 18)
                assert ahead(rows + 1, 1 << 18, 1 << 16, dtype) and not ahead(rows, 1 << 18, 1 << 16, dtype)
