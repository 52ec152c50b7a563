"""Token embedding, dropout and the operators on rows at the ends of their ranges of sizes."""
import ctypes

import pytest
import torch

from lookahead_keys_attention_amd import _native, ops
from test_tokens import kept

DEV = "cuda:0"
gpu = pytest.mark.gpu


@pytest.fixture
def room():
    """room(GiB): skips the test where that much is not free; what it used is given back behind it."""
    def need(gib):
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info()[0] < gib << 30:
            pytest.skip(f"{gib} GiB of the GPU's memory are not free")

    yield need
    if torch.cuda.is_available():
        torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("V", [(1 << 31) - (1 << 26) - 40, (1 << 31) - 2])
def test_the_largest_vocabularies(room, V):
    """Every row of the gradient is written: those of a few tokens, and zeros."""
    room(40)
    table = torch.zeros(V, 1, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    tokens = torch.tensor([0, 5, V - 1, V - 2, V // 2, 5, 1 << 30, V, -1], device=DEV)
    # the memory that the gradient gets holds ones
    stale = torch.ones(V, 1, dtype=torch.bfloat16, device=DEV)
    y = ops.embedding(table, tokens, 2.0)
    assert torch.equal(y.isnan()[:, 0], tokens.eq(V) | tokens.eq(-1))
    dy = torch.arange(1, 10, device=DEV).bfloat16()[:, None]
    del stale
    grad, = torch.autograd.grad(y, table, dy)
    for token, want in ((0, 2), (5, 16), (V - 1, 6), (V - 2, 8), (V // 2, 10), (1 << 30, 14)):
        assert grad[token, 0] == want, token
    assert sum(int(part.count_nonzero()) for part in grad.split(1 << 28)) == 6


@gpu
def test_more_tokens_than_a_launch_has_threads_for(room):
    """2^28 rows of sixteen lanes each are 2^32 threads: the rows behind them, from an index whose rows are the same."""
    room(8)
    table = (torch.arange(1, 1001, device=DEV) / 8).half()[:, None]
    part = torch.randint(0, 1000, (1 << 18,), generator=torch.Generator().manual_seed(1)).to(DEV)
    index = part.expand(1024 + 3, 1 << 18)
    y = ops.embedding(table, index, 2.0)
    assert torch.equal(y[0], (part + 1)[:, None].half() / 4) and bool((y == y[0]).all())


@gpu
def test_dropout_of_more_elements_than_a_launch_has_threads_for(room):
    """2^35 elements, eight to a thread, are 2^32 threads: the mask of the elements around and behind them, on the host."""
    room(140)
    n, p, seed = (1 << 35) + 4099, 0.25, (123456789, 987654321)
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = ops.dropout_add(x, None, p, torch.tensor(seed, device=DEV))
    scale = torch.tensor(65536 / (65536 - round(65536 * p))).bfloat16()
    for first, count in ((0, 1000), ((1 << 34) - 512, 1024), ((1 << 35) - 512, 1024), (n - 1027, 1027)):
        want = torch.where(kept(seed, count, p, first), scale, torch.zeros_like(scale))
        assert torch.equal(y[first:first + count].cpu(), want), first
    for part in y.split(1 << 30):
        assert abs(part.count_nonzero().item() / len(part) - (1 - p)) <= 8 * (p * (1 - p) / len(part)) ** 0.5


@gpu
def test_norm_of_more_rows_than_a_launch_has_threads_for(room):
    """2^28 rows of sixteen lanes each: those behind them are normalised as well."""
    room(16)
    few = torch.randn(1 << 10, 8, generator=torch.Generator().manual_seed(2)).bfloat16().to(DEV)
    x, weight = few.repeat((1 << 18) + 1, 1), torch.full((8,), 0.5, dtype=torch.bfloat16, device=DEV)
    _native.host()
    want = torch.ops.castle_hip.rms_norm(few, weight, 1e-6)
    got = torch.ops.castle_hip.rms_norm(x, weight, 1e-6)
    for a, b in zip(got, want):
        assert bool((a.view(-1, *b.shape) == b).all())


@gpu
def test_gradient_of_the_loss_of_more_rows_than_a_launch_has_threads_for(room):
    """2^26 rows of a wave each."""
    room(12)
    few = torch.randn(1 << 10, 8, generator=torch.Generator().manual_seed(3)).to(DEV)
    logits, n = few.repeat((1 << 16) + 1, 1)[None].requires_grad_(), (1 << 26) + (1 << 10)
    target = torch.arange(n, device=DEV)[None] % 8
    grad, = torch.autograd.grad(_native.host().cross_entropy(logits, target), logits, torch.tensor(float(n), device=DEV))
    want = torch.softmax(few.double(), 1)
    want[range(1 << 10), torch.arange(1 << 10) % 8] -= 1
    # (softmax, the factor and their product in 32 bits, exp with what its argument is off by: 32 steps of 2^-24)
    assert bool(((grad.view(-1, 1 << 10, 8) - want.float()).abs() <= 32 * 2.0 ** -24).all())


@gpu
def test_gradient_without_a_sort_of_a_vocabulary_beyond_the_threads_of_a_launch(room):
    """2^24 rows of the table, a workgroup to each, are 2^32 threads."""
    room(4)
    V, D, tokens = (1 << 24) + 8, 8, torch.tensor([0, 1 << 24, (1 << 24) + 7], device=DEV)
    lib, i, i64, vp = _native.lib(), ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
    size, call = lib.castle_embedding_grad_workspace_bytes, lib.castle_embedding_grad
    size.restype, size.argtypes = i64, [i64, i, i, i]
    call.argtypes = [vp, vp, i64, i64, i64, i, i, vp, i, vp, i64, vp]
    dy, dw = torch.randn(3, D, device=DEV).bfloat16(), torch.ones(V, D, dtype=torch.bfloat16, device=DEV)
    nbytes = size(3, V, D, 1)
    ws = torch.full((nbytes,), 0x3F, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    assert call(dy.data_ptr(), tokens.data_ptr(), 3, 3, 3, V, D, dw.data_ptr(), 1, ws.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream) == 0
    want = torch.zeros_like(dw)
    want[tokens] = dy
    assert torch.equal(dw, want)
