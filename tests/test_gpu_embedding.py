"""Embedding rows and their gradient on the GPU against plain float64 sums.

Tolerances. A looked-up row is one float32 product, off by half a step of float32, and one rounding to its type. A gradient is a float32
sum of t terms in some order: off by at most (t + 8) 2^-24 of the terms' absolute sum S, the product with the scale and the addition to
what was there among the 8.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _tokens(rows, vocabulary, spread, rng, dtype=torch.int32):
    if spread == "even":
        t = rng.integers(0, vocabulary, rows)
    elif spread == "one":
        t = np.full(rows, vocabulary - 1)
    elif spread == "none":
        t = np.where(np.arange(rows) % 2, -1, vocabulary)
    else:                                          # a few tokens in many rows; numbers that are no token on both sides
        t = np.minimum((rng.pareto(0.7, rows) * 2).astype(np.int64), vocabulary + 1) - 1
    return torch.tensor(t, dtype=dtype, device="cuda")


def _wide(t, stride):
    if stride == 1:
        return t
    out = torch.full((t.shape[0], stride, t.shape[1]), float("nan"), dtype=t.dtype, device=t.device)
    out[:, 0] = t
    return out[:, 0]


def _rounding(t):
    return torch.finfo(t).eps / 2


# rows, vocabulary, width, spread, row stride
SHAPES = [(1, 1, 1, "even", 1), (1, 5, 128, "one", 1), (33, 89, 128, "even", 4), (500, 3, 65, "uneven", 1), (257, 1024, 4, "even", 1),
          (700, 1025, 200, "uneven", 2), (300, 40_000, 515, "even", 1), (64, 20, 130, "none", 1), (8192, 70_000, 64, "uneven", 1),
          (8193, 700, 33, "uneven", 3), (9000, 100_003, 96, "even", 1), (30_000, 2, 128, "even", 1), (20_000, 5000, 1032, "uneven", 1),
          (5000, 1, 2500, "one", 1), (12_345, 1_000_000, 7, "uneven", 1), (8191, 1, 40, "one", 1), (8192, 50_000, 40, "uneven", 1), (255, 1_048_575, 3, "even", 1),
          (90, 381, 4096, "uneven", 1)]


@pytest.mark.parametrize("tokens_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", SHAPES)
def test_sorted_tokens(shape, tokens_type):
    from fastmace_b200 import embedding
    rows, vocabulary, _, spread, _ = shape
    t = _tokens(rows, vocabulary, spread, np.random.default_rng(rows), tokens_type)
    order = embedding.sort_tokens(t, vocabulary)
    kept = torch.where((t < 0) | (t >= vocabulary), vocabulary, t).to(torch.int32)
    keys, at = torch.sort(kept, stable=True)
    assert torch.equal(order.keys, keys) and torch.equal(order.rows, at.to(torch.int32))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_and_gradient_against_float64(shape, dtype):
    from fastmace_b200 import embedding
    rows, vocabulary, width, spread, stride = shape
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    t = _tokens(rows, vocabulary, spread, np.random.default_rng(rows + 1), torch.int64 if rows % 2 else torch.int32)
    live = ((t >= 0) & (t < vocabulary)).cpu().numpy()
    at = t.clamp(0, vocabulary - 1).long()
    table = _wide(torch.randn(vocabulary, width, generator=g, device="cuda").to(dtype), stride if vocabulary < 1e5 else 1)
    scale = width ** 0.5
    for out_type in (F32, BF16, F16):
        y = embedding.embedding(t, table, scale, dtype=out_type)
        ref = torch.where(torch.tensor(live, device="cuda")[:, None], table[at].double() * scale, 0.0)
        off = (y.double() - ref).abs()
        # (the scale is rounded to float32 too; a float16 below 2^-14 is half of 2^-24 off)
        assert y.dtype == out_type and bool((off <= (_rounding(out_type) + 2.0 ** -22) * ref.abs() + 2.0 ** -25).all())
    dy = _wide(torch.randn(rows, width, generator=g, device="cuda").to(dtype), stride)
    order = embedding.sort_tokens(t, vocabulary)
    grad = embedding.embedding_gradient(dy, order, vocabulary, scale)
    key = torch.where(torch.tensor(live, device="cuda"), at, vocabulary)
    ref = torch.zeros(vocabulary + 1, width, dtype=torch.float64, device="cuda").index_add_(0, key, dy.double())[:vocabulary] * scale
    size = torch.zeros(vocabulary + 1, width, dtype=torch.float64, device="cuda").index_add_(0, key, dy.double().abs())[:vocabulary] * scale
    count = torch.bincount(key, minlength=vocabulary + 1)[:vocabulary]
    tol = (count[:, None] + 8) * 2.0 ** -24 * size
    assert grad.dtype == F32 and bool(((grad.double() - ref).abs() <= tol).all())
    assert bool((grad[count == 0] == 0).all())
    assert torch.equal(grad, embedding.embedding_gradient(dy, order, vocabulary, scale))          # the same bits again
    base = torch.randn(vocabulary, width, generator=g, device="cuda")
    more = _wide(base.clone(), stride if vocabulary < 1e5 else 1)
    kept = embedding.embedding_gradient(dy, order, vocabulary, scale, out=more, accumulate=True)
    assert kept is more
    assert bool(((more.double() - ref - base.double()).abs() <= (count[:, None] + 9) * 2.0 ** -24 * (size + base.double().abs())).all())
    assert torch.equal(more[count == 0], base[count == 0])


@pytest.mark.parametrize("vocabulary", [1000, 100_003])
def test_millions_of_rows(vocabulary):
    """Sorting CTAs of 32 warps, and a run over more chunks than are looked at together."""
    from fastmace_b200 import embedding
    rows, width = 2_600_000, 8
    g = torch.Generator(device="cuda").manual_seed(vocabulary)
    t = torch.randint(0, vocabulary, (rows,), generator=g, device="cuda")
    t = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.9, 7, t)
    order = embedding.sort_tokens(t, vocabulary)
    keys, at = torch.sort(t, stable=True)
    assert torch.equal(order.keys, keys.to(torch.int32)) and torch.equal(order.rows, at.to(torch.int32))
    dy = torch.randn(rows, width, generator=g, device="cuda")
    grad = embedding.embedding_gradient(dy, order, vocabulary, 0.5)
    total = torch.cat([torch.zeros(1, width, dtype=torch.float64, device="cuda"), dy[at].double().cumsum(0)])
    edge = torch.searchsorted(keys, torch.arange(vocabulary + 1, device="cuda"))
    ref = (total[edge[1:]] - total[edge[:-1]]) * 0.5
    size = torch.cat([torch.zeros(1, width, dtype=torch.float64, device="cuda"), dy[at].double().abs().cumsum(0)])
    size = (size[edge[1:]] - size[edge[:-1]]) * 0.5
    assert bool(((grad.double() - ref).abs() <= ((edge[1:] - edge[:-1])[:, None] + 8) * 2.0 ** -24 * size + 1e-9).all())
    # sums of at most 256 rows a warp, of 8 of those, and of those: the error of the long run is that of far fewer additions in a row
    assert float((grad[7].double() - ref[7]).norm() / size[7].norm()) < 400 * 2.0 ** -24


def test_given_rows_keep_what_no_token_writes():
    from fastmace_b200 import embedding
    t = torch.tensor([2, -1, 0, 3, 2 ** 40], device="cuda")
    table = torch.arange(12, dtype=F32, device="cuda").view(3, 4)
    out = torch.full((5, 4), 7.0, device="cuda")
    embedding.embedding(t, table, 2.0, out=out)
    assert out.tolist() == [[16, 18, 20, 22], [7] * 4, [0, 2, 4, 6], [7] * 4, [7] * 4]
    # a view between other columns: they stay
    wide = torch.full((5, 9), 5.0, device="cuda")
    embedding.embedding(t, table, out=wide[:, 3:7])
    assert bool((wide[:, :3] == 5).all()) and bool((wide[:, 7:] == 5).all()) and wide[0, 3:7].tolist() == [8, 9, 10, 11]
    grad = torch.full((3, 9), 5.0, device="cuda")
    embedding.embedding_gradient(torch.ones(5, 4, device="cuda"), embedding.sort_tokens(t, 3), 3, out=grad[:, 1:5])
    assert grad[:, 1:5].tolist() == [[1] * 4, [0] * 4, [1] * 4] and bool((grad[:, 5:] == 5).all()) and bool((grad[:, 0] == 5).all())


def test_infinities_and_nan_stay_in_their_rows():
    from fastmace_b200 import embedding
    t = torch.tensor([0, 1, 2, 1, -1], device="cuda", dtype=torch.int32)
    dy = torch.ones(5, 40, device="cuda")
    dy[1], dy[2], dy[4] = float("inf"), float("nan"), float("nan")
    grad = embedding.embedding_gradient(dy, embedding.sort_tokens(t, 4), 4)
    assert bool((grad[0] == 1).all()) and bool((grad[1] == float("inf")).all()) and bool(grad[2].isnan().all()) and bool((grad[3] == 0).all())
    table = torch.tensor([[float("nan")] * 8, [1.0] * 8], device="cuda")
    y = embedding.embedding(torch.tensor([1, 5], device="cuda"), table, 3.0)
    assert y.tolist() == [[3.0] * 8, [0.0] * 8]


def test_no_rows():
    from fastmace_b200 import embedding
    t = torch.zeros(0, dtype=torch.int32, device="cuda")
    order = embedding.sort_tokens(t, 7)
    assert embedding.embedding(t, torch.ones(7, 3, device="cuda")).shape == (0, 3)
    grad = torch.ones(7, 3, device="cuda")
    embedding.embedding_gradient(torch.zeros(0, 3, device="cuda"), order, 7, out=grad, accumulate=True)
    assert bool((grad == 1).all())
    assert bool((embedding.embedding_gradient(torch.zeros(0, 3, device="cuda"), order, 7) == 0).all())


def test_captured_and_replayed_on_other_tokens():
    from fastmace_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(5)
    t = torch.randint(0, 3000, (9000,), generator=g, device="cuda")
    table, dy = torch.randn(3000, 48, generator=g, device="cuda"), torch.randn(9000, 48, generator=g, device="cuda")
    run = lambda: (embedding.embedding(t, table, 2.0), embedding.embedding_gradient(dy, embedding.sort_tokens(t, 3000), 3000, 2.0))  # noqa: E731
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            y, grad = run()
    for seed in (6, 7):
        t.copy_(torch.randint(0, 3000, (9000,), generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        again = run()
        assert torch.equal(y, again[0]) and torch.equal(grad, again[1])


def test_gradient_against_differences():
    from fastmace_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(9)
    t = torch.randint(0, 6, (50,), generator=g, device="cuda")
    table, dy = torch.randn(6, 16, generator=g, device="cuda"), torch.randn(50, 16, generator=g, device="cuda")
    step = torch.randn(6, 16, generator=g, device="cuda")
    grad = embedding.embedding_gradient(dy, embedding.sort_tokens(t, 6), 6, 1.5)
    # linear in the table: one difference is exact but for rounding
    loss = lambda w: float((embedding.embedding(t, w, 1.5).double() * dy.double()).sum())  # noqa: E731
    assert abs(loss(table + step) - loss(table) - float((grad.double() * step.double()).sum())) < 1e-3


def test_refusals():
    from fastmace_b200 import embedding
    t, table = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, 8, device="cuda")
    order = embedding.sort_tokens(t, 3)
    dy = torch.zeros(4, 8, device="cuda")
    short = embedding.TokenOrder(order.rows[:3], order.keys[:3])
    nodes = torch.zeros(4, 2, 8, device="cuda")
    for call in (lambda: embedding.sort_tokens(t, 0), lambda: embedding.sort_tokens(t, 1 << 20), lambda: embedding.sort_tokens(t.float(), 3),
                 lambda: embedding.sort_tokens(t[None], 3), lambda: embedding.embedding(t, table.double()),
                 lambda: embedding.embedding(t, table, dtype=torch.float64), lambda: embedding.embedding(t, table.t()),
                 lambda: embedding.embedding(t, table[None]), lambda: embedding.embedding(t, table, out=torch.zeros(3, 8, device="cuda")),
                 lambda: embedding.embedding(t, table, out=torch.zeros(4, 8, device="cuda"), dtype=BF16),
                 lambda: embedding.embedding(t[:3], table, out=table), lambda: embedding.embedding(t.cpu(), table),
                 lambda: embedding.embedding_gradient(dy, short, 3), lambda: embedding.embedding_gradient(dy, order, 3, accumulate=True),
                 lambda: embedding.embedding_gradient(dy.double(), order, 3), lambda: embedding.embedding_gradient(dy, order, 0),
                 lambda: embedding.embedding_gradient(dy, order, 3, out=torch.zeros(2, 8, device="cuda")),
                 lambda: embedding.embedding_gradient(dy, order, 3, out=dy[:3]),
                 lambda: embedding.embedding_gradient(dy, order, 3, out=torch.zeros(3, 8, device="cuda", dtype=BF16)),
                 lambda: embedding.embedding_gradient(nodes[:, 0], order, 4, out=nodes[:, 0])):
        with pytest.raises(ValueError):
            call()
    # two components of one array of features lie apart
    embedding.embedding_gradient(nodes[:, 0], order, 4, out=nodes[:, 1])
