"""Arms of the embedding, routing and expert kernels that other tests' sizes do not reach, against plain float64 evaluations."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _beside(t, extra, front=0):
    """The same rows, with `extra` values between them and `front` before the first."""
    out = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), dtype=t.dtype, device=t.device)
    out[:, front:front + t.shape[1]] = t
    return out[:, front:front + t.shape[1]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocabulary,width", [(40_000, 30, 512), (9000, 5000, 264), (200_000, 89, 128), (30_000, 7, 1024)])
def test_gradient_of_rows_has_the_same_bits_wherever_they_lie(rows, vocabulary, width, dtype):
    from fastmace_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(rows)
    order = embedding.sort_tokens(torch.randint(-1, vocabulary, (rows,), generator=g, device="cuda"), vocabulary)
    dy = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    want = embedding.embedding_gradient(dy, order, vocabulary, 3.0)
    base = torch.randn(vocabulary, width, generator=g, device="cuda")
    more = embedding.embedding_gradient(dy, order, vocabulary, 3.0, out=base.clone(), accumulate=True)
    for extra, front in ((8, 0), (1, 0), (1, 1), (8, 3)):
        view = _beside(dy, extra, front)
        assert torch.equal(embedding.embedding_gradient(view, order, vocabulary, 3.0), want)
        assert torch.equal(embedding.embedding_gradient(view, order, vocabulary, 3.0, out=_beside(base, extra, front), accumulate=True), more)


# rows in a lane's turn: two (rows of 64 packs of a lane's values) and four, aligned and by words and halves, with what is left of rows and columns
@pytest.mark.parametrize("tokens_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocabulary,width,extra,front", [(12_001, 50, 256, 0, 0), (12_001, 50, 512, 0, 0), (12_001, 50, 512, 8, 0), (12_001, 50, 201, 0, 0),
                                                               (12_001, 50, 401, 3, 1), (12_003, 7, 401, 1, 0), (75_777, 50, 33, 2, 1), (10_001, 50, 260, 4, 0)])
def test_rows_side_by_side(rows, vocabulary, width, extra, front, dtype, tokens_type):
    from fastmace_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    table = _beside(torch.randn(vocabulary, width, generator=g, device="cuda").to(dtype), extra, front)
    tokens = torch.randint(-3, vocabulary + 3, (rows,), generator=g, device="cuda", dtype=tokens_type)
    live = ((tokens >= 0) & (tokens < vocabulary))[:, None]
    ref = table[tokens.clamp(0, vocabulary - 1).long()].double() * 0.75
    for out_type in (F32, BF16, F16):
        # one product with a float32 scale, and one rounding (a float16 below 2^-14 is half of 2^-24 off)
        tol = (torch.finfo(out_type).eps / 2 + 2.0 ** -24) * ref.abs() + (2.0 ** -25 if out_type == F16 else 0.0)
        y = embedding.embedding(tokens, table, 0.75, dtype=out_type)
        assert bool(((y.double() - torch.where(live, ref, 0.0)).abs() <= torch.where(live, tol, 0.0)).all())
        held = torch.full((rows, width + extra + 1), 7.0, dtype=out_type, device="cuda")
        embedding.embedding(tokens, table, 0.75, out=held[:, front:front + width])
        assert torch.equal(held[:, front:front + width], torch.where(live, y, 7.0))
        assert bool((held[:, :front] == 7).all()) and bool((held[:, front + width:] == 7).all())


# clusters of two and four tokens, the last ones not full; rows of the router side by side, at other distances and unaligned
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,count,top,width,extra", [(100, 64, 8, 256, 0), (65, 120, 3, 1000, 8), (99, 80, 16, 129, 1), (127, 90, 5, 515, 0),
                                                          (127, 90, 5, 2048, 1), (33, 300, 7, 600, 3), (126, 128, 2, 96, 1)])
def test_routes_of_tokens_that_share_the_router(tokens, count, top, width, extra, dtype, normalise):
    from test_gpu_experts import _check_routes
    g = torch.Generator(device="cuda").manual_seed(tokens + count)
    x = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
    router = (torch.randn(width, count, generator=g, device="cuda") / width ** 0.5).to(dtype)
    _check_routes(x, _beside(router, extra), top, normalise, _beside(x, extra))


# blocks of two, four and eight groups of columns, whose warps are fewer, in the first product and in the second, with groups past the
# matrix's end; what they need is many experts with short depths
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,count,top,width,inner", [(20, 75, 4, 128, 4096), (27, 115, 4, 4096, 128), (64, 256, 8, 100, 1001), (64, 256, 8, 1001, 100),
                                                          (40, 100, 8, 512, 700), (40, 160, 8, 700, 500), (128, 150, 16, 250, 900), (90, 200, 5, 903, 30)])
def test_layers_of_many_experts_and_short_depths(tokens, count, top, width, inner, dtype):
    from fastmace_b200 import experts, grouped
    from test_gpu_experts import _check, _layer
    g = torch.Generator(device="cuda").manual_seed(tokens + width)
    x, up, down = _layer(tokens, count, width, inner, dtype, g)
    chosen = torch.stack([torch.randperm(count, generator=g, device="cuda")[:top] for _ in range(tokens)]).to(torch.int32)
    weights = torch.rand(tokens, top, generator=g, device="cuda")
    routes = experts.Routes(chosen, weights)
    y = experts.expert_layer(x, up, down, routes)
    _check(y, x, up, down, chosen, weights)
    assert torch.equal(y, experts.expert_layer(_beside(x, 1), up, down, routes))
    grouped.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_long_sums_do_not_lose_what_is_small(dtype):
    """A token in 900,000 places: a row of ones in 256, the others below half a step of float32 beside it, so that each is lost where they are added one
    after the other. By eights (3 additions), the eights of a warp's 256 rows (32), the warps of a chunk (8), the 440 chunks by 32 warps (14)
    and those (32) a term goes through 89 additions, each off by half a step of what there is."""
    from fastmace_b200 import embedding
    rows, width = 900_000, 8
    dy = torch.full((rows, width), 63.0 * 2.0 ** -20, device="cuda")
    dy[::256] = 1024.0
    dy = dy.to(dtype)
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    grad = embedding.embedding_gradient(dy, embedding.sort_tokens(tokens, 3), 3)
    want = dy.double().sum(0)
    assert bool(((grad[0].double() - want).abs() <= 89 * 2.0 ** -24 * want).all()), float(((grad[0].double() - want) / want).abs().max() * 2 ** 24)
    assert bool((grad[1:] == 0).all())
