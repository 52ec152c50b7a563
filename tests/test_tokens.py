"""Token embedding of any vocabulary and dropout (ops.embedding, ops.dropout_add): refusals and shapes without a GPU, results against plain forms in 64 bits on one.

Tolerances.  A result is rounded once from sums of 32 bits.  Forward: scale * w is one 32-bit product before it, 2^-24 of the value.  A gradient's element is a sum of n
products with 32-bit additions, n roundings of at most 2^-24 of the sum of the magnitudes, and one product more; the last rounding is at most eps / 2 of the value."""
import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from lookahead_keys_attention_amd import ops

DEV = "cuda:0"
TYPES = [torch.bfloat16, torch.float16, torch.float32]
gpu = pytest.mark.gpu


# ---- plain forms in 64 bits -----------------------------------------------------------------------------------------
def philox(counter, key, at):
    """Philox4x32-10 of the published description, whole numbers on the host -> four words for each counter."""
    mask = (1 << 32) - 1
    out = []
    for n in counter:
        c, k = [n & mask, n >> 32, at & mask, at >> 32 & mask], [key & mask, key >> 32 & mask]
        for _ in range(10):
            p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [q >> 32 ^ c[1] ^ k[0], q & mask, p >> 32 ^ c[3] ^ k[1], p & mask]
            k = [k[0] + 0x9E3779B9 & mask, k[1] + 0xBB67AE85 & mask]
        out.append(c)
    return out


def kept(seed, n, p, first=0):
    """Whether elements first ... first + n - 1 stay; `first` a multiple of 8."""
    words = philox(range(first // 8, (first + n + 7) // 8), seed[0] % 2 ** 64, seed[1] % 2 ** 64)
    halves = [h for group in words for w in group for h in (w & 0xFFFF, w >> 16)][:n]
    return torch.tensor([h >= round(65536 * p) for h in halves])


def dropped(x, residual, seed, p):
    t = round(65536 * p)
    keep = kept(seed, x.numel(), p).view(x.shape)
    y = torch.where(keep, x.double() * (65536 / (65536 - t) if t < 65536 else 0), 0.0)
    return y if residual is None else y + residual.double()


def table_grad(dy, index, V, scale, padding):
    """(gradient, sum of the magnitudes, number of summands) in 64 bits."""
    d, t = dy.double().reshape(-1, dy.shape[-1]), index.reshape(-1).long()
    there = (t >= 0) & (t < V) & (t != (-1 if padding is None else padding))
    d, t = d[there], t[there]
    sums = torch.zeros(V, dy.shape[-1], dtype=torch.float64)
    return (sums.index_add(0, t, d) * scale, sums.index_add(0, t, d.abs()) * abs(scale),
            torch.zeros(V, 1, dtype=torch.float64).index_add(0, t, torch.ones(len(t), 1, dtype=torch.float64)))


def within(got, ref, slack, dtype, what):
    got, ref = got.detach().cpu().double(), ref.double()
    assert torch.equal(got.isfinite(), ref.isfinite()), what
    # half a step of the type, of the value or of the smallest normal number
    half = torch.finfo(dtype).eps / 2
    most = slack + half * (ref.abs() + slack).clamp(min=torch.finfo(dtype).tiny)
    off = (got - ref).abs()
    assert (off <= most).all(), (what, (off - most).max())


# ---- without a GPU --------------------------------------------------------------------------------------------------
def test_philox_of_the_published_vectors():
    """The test vectors that the generator's authors publish with it: zeros, and all ones."""
    assert philox([0], 0, 0) == [[0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]]
    ones = 2 ** 64 - 1
    assert philox([ones], ones, ones) == [[0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]]


def test_operators_trace_and_keep_shapes():
    with FakeTensorMode():
        w = torch.empty(50, 12, dtype=torch.bfloat16, requires_grad=True)
        y = ops.embedding(w, torch.zeros(3, 4, dtype=torch.long), 2.0, 7)
        assert y.shape == (3, 4, 12) and y.dtype == torch.bfloat16
        y.sum().backward()
        assert w.grad.shape == w.shape
        x, r = torch.empty(3, 5, requires_grad=True), torch.empty(3, 5, requires_grad=True)
        ops.dropout_add(x, r, 0.5, torch.zeros(2, dtype=torch.long)).sum().backward()
        assert x.grad.shape == r.grad.shape == x.shape
        grad, = torch.autograd.grad(ops.embedding(w, torch.zeros(3, dtype=torch.long)).float().square().sum(), w, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            grad.sum().backward()
    for name in ("embedding", "embedding_bwd", "dropout_add"):
        assert "!" not in str(getattr(torch.ops.castle_hip, name).default._schema)   # functional


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(RuntimeError, match="GPU"):
        ops.embedding(torch.zeros(4, 8), torch.zeros(3, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.dropout_add(torch.zeros(8), None, 0.1, torch.zeros(2, dtype=torch.long))
    for bad in (-1, 4):
        with pytest.raises(ValueError):
            ops.embedding(torch.zeros(4, 8), torch.zeros(3, dtype=torch.long), padding_idx=bad)


def test_entry_points_check_their_arguments_on_the_host():
    import ctypes

    from lookahead_keys_attention_amd import _native as N

    lib, i, i64, f, d, vp = N.lib(), ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double, ctypes.c_void_p
    size = lib.castle_embedding_sorted_grad_workspace_bytes
    size.restype, size.argtypes = i64, [i64, i, i]
    assert size(0, 10, 8) == size(5, 0, 8) == size(5, 10, 0) == size((1 << 30) + 1, 10, 8) == size(5, 2 ** 31 - 1, 8) == -2
    for rows, V, D in ((1, 1, 1), (63, 300, 7), (70000, 131072, 64), (1 << 22, 1000, 8)):
        # two sorts' worth of keys and places, and a row of floats for each 64 tokens
        assert 16 * rows + rows // 64 * D * 4 <= size(rows, V, D) <= 16 * rows + rows // 64 * D * 4 + (2 << 20)
    p = 4096
    emb = lib.castle_embedding
    emb.argtypes = [vp, i64, i, i, vp, i64, i64, i64, f, vp, i, vp]
    good = [p, 8, 10, 8, p, 6, 6, 6, 1.0, p, 1, None]
    for at, bad, code in ((10, 3, -1), (2, 0, -2), (3, 0, -2), (5, 4, -2), (7, 0, -2), (7, (1 << 30) + 6, -2), (0, None, -5), (0, p + 1, -5), (4, p + 4, -5), (9, p + 1, -5), (1, -8, -5), (6, -6, -5)):
        args = list(good)
        args[at] = bad
        assert emb(*args) == code, (at, bad)
    grad = lib.castle_embedding_sorted_grad
    grad.argtypes = [vp, vp, i64, i64, i64, i, i, f, i, vp, i, vp, i64, vp]
    good = [p, p, 6, 6, 6, 10, 8, 1.0, -1, p, 1, p, 1 << 30, None]
    for at, bad, code in ((10, 7, -1), (2, 4, -2), (4, 0, -2), (5, 0, -2), (0, p + 1, -5), (1, None, -5), (9, None, -5), (8, 10, -5), (8, -2, -5), (3, -1, -5), (11, None, -4), (11, p + 16, -4), (12, 100, -4)):
        args = list(good)
        args[at] = bad
        assert grad(*args) == code, (at, bad)
    drop = lib.castle_dropout
    drop.argtypes = [vp, vp, vp, i64, d, vp, i, vp]
    good = [p, None, p, 100, 0.1, p, 1, None]
    for at, bad, code in ((6, 9, -1), (3, 0, -2), (3, (1 << 40) + 1, -2), (0, None, -5), (1, p + 8, -5), (2, p + 2, -5), (4, -0.1, -5), (4, 1.5, -5), (4, float("nan"), -5), (5, p + 4, -5)):
        args = list(good)
        args[at] = bad
        assert drop(*args) == code, (at, bad)


# ---- embedding ------------------------------------------------------------------------------------------------------
def check_embedding(w, index, dy, scale, padding=None):
    V, dtype = w.shape[0], w.dtype
    leaf = w.to(DEV).requires_grad_()
    y = ops.embedding(leaf, index.to(DEV), scale, padding)
    there = (index >= 0) & (index < V)
    ref = torch.where(there[..., None], w.double()[index.long().clamp(0, V - 1)] * scale, float("nan"))
    assert torch.equal(y.isnan().cpu(), ref.isnan())
    within(y.cpu()[there], ref[there], 2.0 ** -24 * ref[there].abs(), dtype, "y")
    got, = torch.autograd.grad(y, leaf, dy.to(DEV))
    ref, magnitude, n = table_grad(dy, index, V, scale, padding)
    within(got, ref, (n + 1) * 2.0 ** -24 * magnitude, dtype, "gradient")
    return got


# one token to several workgroups of the sort; widths of pieces and of none, of one lane and of several rounds; vocabularies of one, two and three digits
@gpu
@pytest.mark.parametrize("V,D,B,n", [(1, 8, 1, 1), (5, 1, 2, 33), (300, 7, 3, 64), (300, 128, 1, 65), (1023, 250, 2, 700), (1024, 512, 3, 683), (32000, 64, 4, 1500),
                                     (50257, 24, 1, 4097), (131072, 16, 2, 9000), (1 << 20, 8, 2, 500), (2000, 2056, 1, 300)])
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_and_its_gradient(V, D, B, n, dtype):
    g = torch.Generator().manual_seed(V + D)
    w = torch.randn(V, D, generator=g).to(dtype)
    ids = (torch.rand(B, n + 1, generator=g, dtype=torch.float64) * np.log(V + 1)).exp().long().sub(1).clamp(0, V - 1)
    dy = torch.randn(B, n, D, generator=g).to(dtype)
    check_embedding(w, ids[:, :-1], dy, D ** 0.5, 0 if V > 1 and n > 60 else None)


@gpu
@pytest.mark.parametrize("n", [8, 9, 63, 64, 65, 127, 128, 129, 200, 1000])
def test_gradient_of_one_token_again_and_again(n):
    """Runs of one token from every place to every place of a piece of 64, alone and between others."""
    g = torch.Generator().manual_seed(n)
    w = torch.randn(40, 40, generator=g)
    for before in (0, 1, 63, 64, 100):
        ids = torch.cat((torch.full((before,), 3), torch.full((n,), 17), torch.full((70,), 39)))[torch.randperm(before + n + 70, generator=g)]
        check_embedding(w, ids, torch.randn(len(ids), 40, generator=g), 1.0)


@gpu
@pytest.mark.parametrize("V", [255, 256, 511, 512, 65535, 65536, (1 << 18) - 1, 1 << 18])
@pytest.mark.parametrize("n", [1, 1023, 8191, 8192, 8193, 16385])
def test_gradient_where_the_sorting_changes(n, V):
    """Whole numbers, whose sums are exact in 32 bits: every token in its row, at the digits and numbers of tokens where another way of sorting begins."""
    g = torch.Generator().manual_seed(n + V)
    w = torch.zeros(V, 4)
    ids = (torch.rand(n, generator=g, dtype=torch.float64) * np.log(V + 1)).exp().long().sub(1).clamp(0, V - 1)
    ids[-1] = V - 1
    dy = torch.randint(-8, 9, (n, 4), generator=g).float()
    leaf = w.to(DEV).requires_grad_()
    ops.embedding(leaf, ids.to(DEV)).backward(dy.to(DEV))
    assert torch.equal(leaf.grad.cpu(), w.index_add(0, ids, dy))


@gpu
def test_embedding_tokens_that_are_not_there_and_masked_values():
    g = torch.Generator().manual_seed(1)
    w, ids = torch.randn(100, 16, generator=g), torch.randint(0, 100, (4, 50), generator=g)
    ids[0, :9] = torch.tensor([-1, 100, 1 << 40, -(1 << 40), -100, 1 << 32, (1 << 32) + 5, 2 ** 63 - 1, -2 ** 63])
    ids[1] = 7
    dy = torch.randn(4, 50, 16, generator=g)
    dy[0, :9], dy[1] = float("nan"), float("inf")   # tokens outside, and padding
    grad = check_embedding(w, ids, dy, 3.0, 7)
    assert grad.isfinite().all() and not grad[7].any()
    # no token at all
    all_out = torch.full((3, 5), 100)
    assert not check_embedding(w, all_out, torch.randn(3, 5, 16, generator=g), 1.0).any()


@gpu
def test_embedding_of_other_layouts():
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(60, 48, generator=g).bfloat16()
    ids = torch.randint(0, 60, (6, 4, 7), generator=g)
    dy = torch.randn(6, 4, 7, 20, generator=g).bfloat16()
    table = wide.to(DEV)[:, 4:24].detach().requires_grad_()   # rows of a wider table, not at 16 bytes
    index = ids.to(DEV).permute(2, 0, 1)
    y = ops.embedding(table, index, 0.5)
    assert y.shape == (7, 6, 4, 20) and torch.equal(y.cpu(), (wide[:, 4:24][ids.permute(2, 0, 1)].float() * 0.5).bfloat16())
    y.backward(dy.to(DEV).permute(2, 0, 1, 3))
    ref, magnitude, n = table_grad(dy.permute(2, 0, 1, 3), ids.permute(2, 0, 1), 60, 0.5, None)
    within(table.grad, ref, (n + 1) * 2.0 ** -24 * magnitude, torch.bfloat16, "gradient")
    transposed = wide.to(DEV).t()   # (48, 60), columns contiguous
    assert torch.equal(ops.embedding(transposed, ids.to(DEV).int() % 48), transposed.contiguous()[ids.to(DEV) % 48])
    assert ops.embedding(table, torch.zeros(0, 3, dtype=torch.long, device=DEV)).shape == (0, 3, 20)
    grad, = torch.autograd.grad(ops.embedding(table, torch.zeros(0, dtype=torch.long, device=DEV)).sum(), table)
    assert grad.shape == table.shape and not grad.any()
    for bad in (lambda: ops.embedding(table.double(), index), lambda: ops.embedding(table, index.float()), lambda: ops.embedding(table, index.cpu()),
                lambda: ops.embedding(table[0], index), lambda: ops.embedding(table[:0], index)):
        with pytest.raises((TypeError, ValueError)):
            bad()


@gpu
def test_embedding_gradient_is_the_same_every_time_in_graphs_and_on_other_streams():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(3000, 64, generator=g).to(DEV).requires_grad_()
    ids, dy = torch.randint(0, 3000, (5, 2000), generator=g).to(DEV) % 700, torch.randn(5, 2000, 64, generator=g).to(DEV)

    def step():
        return torch.autograd.grad(ops.embedding(w, ids, 2.0), w, dy)[0]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(step(), want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        ids.copy_(ids.flip(1) if k else ids)
        dy.mul_(1 if k == 0 else -1)
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


@gpu
def test_embedding_of_a_table_past_32_bits_of_elements():
    V, D = 70001, 65536
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(4)
    few = torch.tensor([0, 1, 32768, 65535, 65536, 65537, V - 1])
    rows = torch.randn(len(few), D, generator=g).bfloat16().to(DEV)
    w[few.to(DEV)] = rows
    ids = torch.randint(0, len(few), (90,), generator=g)
    dy = torch.randint(-8, 9, (90, D), generator=g).bfloat16().to(DEV)   # (whole numbers: exact sums)
    y = ops.embedding(w.requires_grad_(), few[ids].to(DEV), 2.0)
    assert torch.equal(y, 2 * rows[ids.to(DEV)])
    grad, = torch.autograd.grad(y, w, dy)
    want = torch.zeros(len(few), D, device=DEV).index_add_(0, ids.to(DEV), 2 * dy.float())
    assert torch.equal(grad[few.to(DEV)], want.bfloat16())
    grad[few.to(DEV)] = 0
    assert grad.count_nonzero() == 0


# ---- dropout --------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (3, 333, 5), (2, 1024, 16), (4100,)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9, 1.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_with_and_without_a_residual(shape, p, dtype):
    g = torch.Generator().manual_seed(len(shape))
    seed = torch.randint(-2 ** 63, 2 ** 63 - 1, (2,), generator=g)
    x, r, dy = (torch.randn(shape, generator=g).to(dtype) for _ in range(3))
    for residual in (None, r):
        leaves = [t.to(DEV).requires_grad_() for t in (x, r)]
        y = ops.dropout_add(leaves[0], leaves[1] if residual is not None else None, p, seed.to(DEV))
        ref = dropped(x, residual, seed.tolist(), p)
        # a product and a sum of 32 bits before the rounding
        within(y, ref, 2.0 ** -23 * (ref.abs() + (0 if residual is None else residual.double().abs())), dtype, "y")
        y.backward(dy.to(DEV))
        within(leaves[0].grad, dropped(dy, None, seed.tolist(), p), 2.0 ** -23 * dy.double().abs() * (1 / (1 - p) if p < 1 else 0), dtype, "dx")
        if residual is not None:
            assert torch.equal(leaves[1].grad.cpu(), dy)


@gpu
def test_dropout_leaves_nothing_of_what_it_drops_and_refuses_what_it_cannot_do():
    seed = torch.tensor([5, 6], device=DEV)
    for bad in (float("nan"), float("inf")):
        x = torch.full((1000,), bad, device=DEV)
        y = ops.dropout_add(x, torch.ones_like(x), 0.5, seed)
        assert torch.equal((y == 1).cpu(), ~kept((5, 6), 1000, 0.5))
    # other numbers, another mask; about as many as asked for: 8000 draws, six standard deviations
    ones = torch.ones(8000, device=DEV)
    masks = [ops.dropout_add(ones, None, 0.25, torch.tensor(s, device=DEV)) != 0 for s in ((1, 0), (2, 0), (1, 1), (1 + (1 << 32), 0), (1, 1 << 32))]
    for i, a in enumerate(masks):
        assert abs(a.sum().item() - 6000) < 6 * (8000 * 0.25 * 0.75) ** 0.5
        assert all(not torch.equal(a, b) for b in masks[:i])
    x = torch.randn(30, 40, device=DEV)
    assert torch.equal(ops.dropout_add(x.t(), None, 0.3, seed), ops.dropout_add(x.t().contiguous(), None, 0.3, seed))
    assert torch.equal(ops.dropout_add(x.flatten()[1:], None, 0.3, seed), ops.dropout_add(x.flatten()[1:].clone(), None, 0.3, seed))
    assert ops.dropout_add(x[:0], None, 0.3, seed).shape == (0, 40)
    for bad in (lambda: ops.dropout_add(x, None, -0.1, seed), lambda: ops.dropout_add(x, None, 1.1, seed), lambda: ops.dropout_add(x, None, float("nan"), seed),
                lambda: ops.dropout_add(x, x[:1], 0.1, seed), lambda: ops.dropout_add(x, x.half(), 0.1, seed), lambda: ops.dropout_add(x, None, 0.1, seed[:1]),
                lambda: ops.dropout_add(x, None, 0.1, seed.cpu()), lambda: ops.dropout_add(x, None, 0.1, seed.int()), lambda: ops.dropout_add(x.double(), None, 0.1, seed)):
        with pytest.raises((TypeError, ValueError)):
            bad()


@gpu
def test_dropout_counters_past_32_bits_of_elements():
    """An element behind 2^32 of them (2^29 groups of eight still fit a word; the place of an element does not)."""
    n = (1 << 32) + 24
    x = torch.ones(n, device=DEV, dtype=torch.bfloat16)
    y = ops.dropout_add(x, None, 0.5, torch.tensor([9, 10], device=DEV))
    assert torch.equal((y[-24:] != 0).cpu(), kept((9, 10), 24, 0.5, first=1 << 32))
    assert torch.equal((y[:64] != 0).cpu(), kept((9, 10), 64, 0.5))


@gpu
def test_dropout_in_a_graph_reads_its_numbers_anew():
    x, dy = torch.randn(5, 1000, device=DEV, requires_grad=True), torch.randn(5, 1000, device=DEV)
    seed = torch.tensor([1, 2], device=DEV)

    def step():
        y = ops.dropout_add(x, x, 0.3, seed)
        return y, torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    last = None
    for k in range(4):
        seed.copy_(torch.tensor([k, 7 * k], device=DEV))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert last is None or not torch.equal(last, got[0])
        last = got[0].clone()


@gpu
def test_opcheck():
    g = torch.Generator().manual_seed(0)
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    w, ids = torch.randn(30, 8, generator=g).to(DEV).requires_grad_(), torch.randint(0, 30, (4, 5), generator=g).to(DEV)
    torch.library.opcheck(torch.ops.castle_hip.embedding.default, (w, ids, 2.0, -1), test_utils=tests)
    x, seed = torch.randn(3, 5, generator=g).to(DEV).requires_grad_(), torch.tensor([1, 2], device=DEV)
    torch.library.opcheck(torch.ops.castle_hip.dropout_add.default, (x, x, 0.3, seed), test_utils=tests)
