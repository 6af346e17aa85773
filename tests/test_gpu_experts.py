"""Routing and the expert layer for a few tokens on the GPU against plain float64 evaluations.

Tolerances. A float32 sum of t products is off by (t + 8) 2^-24 of the terms' absolute sum S; float32 operands are 22 bits of each factor and the
smallest of four products is left out, 2^-20 S more. h = silu(a) b is off by 1.1 |b| da + |silu(a)| db (the slope of silu is below 1.1) and by
its own roundings, 2^-20 of itself; between the products it keeps 17 bits at least: 2^-16. y is the weighted sum of that, and rounded once.
Logits are float32 sums; the inputs of the tests have gaps between logits far above their errors, or exact ties.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _wide(t, stride):
    if stride == 1:
        return t
    out = torch.full((t.shape[0], stride, t.shape[1]), float("nan"), dtype=t.dtype, device=t.device)
    out[:, 0] = t
    return out[:, 0]


def _layer(t, experts, width, inner, dtype, g):
    x = torch.randn(t, width, generator=g, device="cuda").to(dtype)
    up = (torch.randn(experts, width, 2 * inner, generator=g, device="cuda") / width ** 0.5).to(dtype)
    down = (torch.randn(experts, inner, width, generator=g, device="cuda") / inner ** 0.5).to(dtype)
    return x, up, down


def _reference(x, up, down, chosen, weights):
    """(y, how far it may be off before its rounding) in float64."""
    y, off = torch.zeros(x.shape, dtype=torch.float64, device="cuda"), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    experts, width, inner = up.shape[0], up.shape[1], down.shape[1]
    more = 2.0 ** -20 if x.dtype == F32 else 0.0
    for e in range(experts):
        t, j = torch.nonzero(chosen == e, as_tuple=True)
        if not len(t):
            continue
        xs, wu, wd, w = x[t].double(), up[e].double(), down[e].double(), weights[t, j].double()[:, None]
        u, size = xs @ wu, xs.abs() @ wu.abs()
        (a, b), (da, db) = u.chunk(2, 1), (size * ((width + 8) * 2.0 ** -24 + more)).chunk(2, 1)
        silu = a / (1 + torch.exp(-a))
        h = silu * b
        dh = 1.1 * b.abs() * da + silu.abs() * db + da * db + h.abs() * (2.0 ** -20 + 2.0 ** -16)
        y.index_add_(0, t, w * (h @ wd))
        off.index_add_(0, t, w.abs() * (dh @ wd.abs() + ((inner + 8) * 2.0 ** -24 + more) * (h.abs() @ wd.abs())))
    return y, off + 2.0 ** -22 * y.abs() + chosen.shape[1] * 2.0 ** -24 * off


def _check(y, x, up, down, chosen, weights):
    ref, off = _reference(x, up, down, chosen, weights)
    half = torch.finfo(y.dtype).eps / 2
    assert y.dtype == x.dtype
    far = (y.double() - ref).abs() - off - half * (ref.abs() + off) - (2.0 ** -25 if y.dtype == F16 else 0.0)
    assert bool((far <= 0).all()), (float(far.max()), float((y.double() - ref).norm() / ref.norm()))


# tokens, experts, top, width, inner, row stride
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 8, 2, 64, 32, 1), (1, 64, 8, 256, 128, 1), (3, 5, 5, 33, 17, 2), (8, 1, 1, 128, 96, 1), (9, 4, 2, 130, 70, 1),
          (16, 3, 2, 264, 136, 3), (33, 40, 3, 101, 55, 1), (64, 4, 2, 512, 256, 1), (128, 2, 1, 72, 40, 1), (128, 200, 16, 64, 64, 1),
          (17, 1024, 4, 40, 24, 1), (2, 6, 3, 2056, 1032, 1), (5, 3, 2, 1024, 4100, 1), (100, 1, 1, 65, 31, 1)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer_against_float64(shape, dtype):
    from fastmace_b200 import experts, grouped
    t, count, top, width, inner, stride = shape
    g = torch.Generator(device="cuda").manual_seed(t + width)
    x, up, down = _layer(t, count, width, inner, dtype, g)
    chosen = torch.stack([torch.randperm(count, generator=g, device="cuda")[:top] for _ in range(t)]).to(torch.int32)
    weights = torch.rand(t, top, generator=g, device="cuda")
    routes = experts.Routes(chosen, weights)
    y = experts.expert_layer(_wide(x, stride), up, down, routes)
    _check(y, x, up, down, chosen, weights)
    assert torch.equal(y, experts.expert_layer(x, up, down, routes))                     # the same bits again
    others, elsewhere = torch.randn(x.shape, generator=g, device="cuda").to(dtype), torch.roll(chosen, 1, 0)
    others[t - 1], elsewhere[t - 1] = x[t - 1], chosen[t - 1]
    one = experts.expert_layer(others, up, down, experts.Routes(elsewhere, weights))
    assert torch.equal(one[t - 1], y[t - 1])                                              # whatever the other tokens are
    given = torch.full((t, 3, width), 7.0, device="cuda", dtype=dtype)
    experts.expert_layer(x, up, down, routes, out=given[:, 1])
    assert torch.equal(given[:, 1], y) and bool((given[:, 0] == 7).all()) and bool((given[:, 2] == 7).all())
    grouped.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_choices_that_are_no_expert_or_alike(dtype):
    from fastmace_b200 import experts
    g = torch.Generator(device="cuda").manual_seed(1)
    x, up, down = _layer(40, 6, 96, 48, dtype, g)
    chosen = torch.randint(-2, 8, (40, 4), generator=g, device="cuda", dtype=torch.int32)
    chosen[0], chosen[1], chosen[2] = -1, 2 ** 31 - 1, 3              # nothing, nothing, the same expert four times
    weights = torch.randn(40, 4, generator=g, device="cuda")
    y = experts.expert_layer(x, up, down, experts.Routes(chosen, weights))
    _check(y, x, up, down, chosen, weights)
    assert bool((y[:2] == 0).all())
    assert bool((experts.expert_layer(x, up, down, experts.Routes(torch.full_like(chosen, -1), weights)) == 0).all())
    # all rows at one expert: more than a unit takes at a time
    chosen = torch.full((40, 4), 5, dtype=torch.int32, device="cuda")
    _check(experts.expert_layer(x, up, down, experts.Routes(chosen, weights)), x, up, down, chosen, weights)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_views_of_weights(dtype):
    from fastmace_b200 import experts
    g = torch.Generator(device="cuda").manual_seed(2)
    x, up, down = _layer(5, 3, 40, 24, dtype, g)
    chosen, weights = torch.tensor([[0, 2], [1, 0], [2, 1], [0, 1], [1, 2]], device="cuda", dtype=torch.int32), torch.rand(5, 2, generator=g, device="cuda")
    want = experts.expert_layer(x, up, down, experts.Routes(chosen, weights))
    big = torch.full((40, 3, 60), float("nan"), device="cuda", dtype=dtype)
    big[:, :, 5:53] = up.permute(1, 0, 2)
    wide = torch.full((3, 24, 48), float("nan"), device="cuda", dtype=dtype)
    wide[:, :, 8:] = down
    got = experts.expert_layer(x, big[:, :, 5:53].permute(1, 0, 2), wide[:, :, 8:], experts.Routes(chosen, weights))
    assert torch.equal(got, want)


def test_large_values_between_the_products():
    """float16 weights: what passes the gate may be beyond float16's range."""
    from fastmace_b200 import experts
    for dtype, big in ((F16, 600.0), (BF16, 1e6), (F32, 1e8)):
        x = torch.full((1, 64), 1.0, device="cuda", dtype=dtype)
        up = torch.full((1, 64, 32), big / 64, device="cuda", dtype=dtype)
        down = torch.full((1, 16, 64), 2.0 ** -14, device="cuda", dtype=dtype)
        y = experts.expert_layer(x, up, down, experts.Routes(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda")))
        u = float(up[0, 0, 0]) * 64
        assert bool(((y.double() / (16 * u * u * 2.0 ** -14) - 1).abs() < torch.finfo(dtype).eps + 2.0 ** -15).all())


def test_infinities_and_nan_stay_with_their_tokens():
    from fastmace_b200 import experts
    g = torch.Generator(device="cuda").manual_seed(4)
    for dtype in (F32, BF16, F16):
        x, up, down = _layer(12, 2, 64, 32, dtype, g)
        routes = experts.Routes(torch.zeros(12, 1, dtype=torch.int32, device="cuda"), torch.ones(12, 1, device="cuda"))
        want = experts.expert_layer(x, up, down, routes)
        bad = x.clone()
        bad[3], bad[9, 5] = float("nan"), float("inf")
        y = experts.expert_layer(bad, up, down, routes)
        keep = [i for i in range(12) if i not in (3, 9)]
        assert torch.equal(y[keep], want[keep]) and bool(y[3].isnan().all()) and not bool(y[9].isfinite().any())


def _check_routes(x, router, top, normalise, given):
    from fastmace_b200 import experts
    (t, width), count = x.shape, router.shape[1]
    routes = experts.route_rows(given, router, top, normalise)
    logits, size = x.double() @ router.double(), x.double().abs() @ router.double().abs()
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
    got = torch.gather(logits, 1, routes.experts.long())
    # sums in float32: width additions of half a step, and what the tensor core cuts off
    tol = (width + 8) * 2.0 ** -24 * size.amax(1, keepdim=True)
    assert bool(((got - torch.gather(logits, 1, order)).abs() <= 2 * tol).all())
    assert all(len(set(row)) == top for row in routes.experts.tolist())
    p = torch.softmax(got if normalise else logits, 1)
    p = p if normalise else torch.gather(p, 1, routes.experts.long())
    assert bool(((routes.weights.double() - p).abs() <= p * (4 * tol + (count + 16) * 2.0 ** -24) + 1e-30).all())
    again = experts.route_rows(x.contiguous(), router, top, normalise)
    assert torch.equal(again.experts, routes.experts) and torch.equal(again.weights, routes.weights)


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(129, 64, 8, 64), (130, 300, 16, 192), (257, 1024, 4, 72), (3, 1000, 5, 2000), (4097, 65, 5, 520), (140, 256, 16, 1),
                                   (150, 9, 2, 4096), (129, 128, 1, 63), (10001, 17, 3, 129), (128, 250, 8, 1000), (40000, 8, 2, 96)])
def test_routes_of_many_tokens(shape, dtype, normalise):
    t, count, top, width = shape
    g = torch.Generator(device="cuda").manual_seed(t + count)
    x = torch.randn(t, width, generator=g, device="cuda").to(dtype)
    router = (torch.randn(width, count, generator=g, device="cuda") / width ** 0.5).to(dtype)
    for extra in (0, 3, 8):                  # rows side by side, odd and at whole pieces of 16 bytes
        held = [torch.full((m.shape[0], m.shape[1] + extra), float("nan"), dtype=dtype, device="cuda") for m in (x, router)]
        for h, m in zip(held, (x, router)):
            h[:, :m.shape[1]] = m
        _check_routes(x, held[1][:, :count], top, normalise, held[0][:, :width])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [130, 20000])
def test_routes_of_many_tokens_with_equal_and_bad_logits(dtype, tokens):
    from fastmace_b200 import experts
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(tokens, 64, device="cuda", dtype=dtype)
    x[:, 0] = 1
    router = torch.zeros(64, 70, device="cuda", dtype=dtype)
    router[0] = torch.tensor([1.0, -0.0, 0.0, 2.0, 1.0, 2.0] + [0.5] * 64, device="cuda").to(dtype)
    routes = experts.route_rows(x, router, 6)
    assert bool((routes.experts == torch.tensor([3, 5, 0, 4, 6, 7], device="cuda")).all())
    router[0, 3], router[0, 9] = nan, -inf       # infinities times the zeros of x are nowhere else
    routes = experts.route_rows(x, router, 6)
    assert bool((routes.experts == torch.tensor([5, 0, 4, 6, 7, 8], device="cuda")).all()) and bool(routes.weights.isfinite().all())
    assert bool(experts.route_rows(x, router, 6, normalise=False).weights.isnan().all())
    # one bad token: its own row alone
    router[0, 3] = 2.0
    want = experts.route_rows(x, router, 6)
    x[77] = nan
    routes = experts.route_rows(x, router, 6)
    assert routes.experts[77].tolist() == [0, 1, 2, 3, 4, 5] and bool(routes.weights[77].isnan().all())
    rest = torch.arange(tokens, device="cuda") != 77
    assert torch.equal(routes.experts[rest], want.experts[rest]) and torch.equal(routes.weights[rest], want.weights[rest])
    # all choices are NaN, in their order
    router[0] = nan
    assert bool((experts.route_rows(x, router, 6).experts == torch.arange(6, device="cuda")).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [300, 12000])
def test_routes_of_many_tokens_captured_and_on_two_streams(tokens, dtype):
    from fastmace_b200 import experts
    g = torch.Generator(device="cuda").manual_seed(tokens)
    xs = [torch.randn(tokens, 520, generator=g, device="cuda").to(dtype) for _ in range(4)]
    router = torch.randn(520, 130, generator=g, device="cuda").to(dtype)
    want = [experts.route_rows(x, router, 6) for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = experts.route_rows(x, router, 6)
    for given, routes in zip(xs, want):
        x.copy_(given)
        graph.replay()
        assert torch.equal(held.experts, routes.experts) and torch.equal(held.weights, routes.weights)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for n, given in enumerate(xs):
        with torch.cuda.stream(streams[n % 2]):
            got.append(experts.route_rows(given, router, 6))
    torch.cuda.synchronize()
    assert all(torch.equal(a.experts, b.experts) and torch.equal(a.weights, b.weights) for a, b in zip(got, want))


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (3, 64, 8, 256), (40, 7, 7, 65), (200, 40, 3, 1001), (5, 1024, 16, 128), (2, 9, 2, 4096), (1000, 128, 8, 64)])
def test_routes_against_float64(shape, dtype, normalise):
    from fastmace_b200 import experts
    t, count, top, width = shape
    g = torch.Generator(device="cuda").manual_seed(t + count)
    x = torch.randn(t, width, generator=g, device="cuda").to(dtype)
    router = (torch.randn(width, count, generator=g, device="cuda") / width ** 0.5).to(dtype)
    routes = experts.route_rows(_wide(x, 2), router, top, normalise)
    logits, size = x.double() @ router.double(), x.double().abs() @ router.double().abs()
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
    got = torch.gather(logits, 1, routes.experts.long())
    tol = (width + 8) * 2.0 ** -24 * size.amax(1, keepdim=True)
    # the same choices, but for logits that are nearer than their errors
    assert bool(((got - torch.gather(logits, 1, order)).abs() <= 2 * tol).all())
    assert float((routes.experts == order).double().mean()) > 0.999
    assert all(len(set(row)) == top for row in routes.experts.tolist())
    p = torch.softmax(got if normalise else logits, 1)
    p = p if normalise else torch.gather(p, 1, routes.experts.long())
    assert bool(((routes.weights.double() - p).abs() <= p * (4 * tol + (count + 16) * 2.0 ** -24) + 1e-30).all())
    again = experts.route_rows(x, router, top, normalise)
    assert torch.equal(again.experts, routes.experts) and torch.equal(again.weights, routes.weights)


def test_equal_logits_go_by_number_and_nan_comes_last():
    from fastmace_b200 import experts
    x = torch.ones(3, 8, device="cuda")
    router = torch.zeros(8, 70, device="cuda")
    router[0] = torch.tensor([1.0, -0.0, 0.0, 2.0, 1.0, 2.0] + [0.5] * 64, device="cuda")
    assert experts.route_rows(x, router, 6).experts[1].tolist() == [3, 5, 0, 4, 6, 7]
    router[0, 3] = float("nan")
    assert experts.route_rows(x, router, 6).experts[2].tolist() == [5, 0, 4, 6, 7, 8]
    small = router[:, :4].contiguous()
    routes = experts.route_rows(x, small, 4)
    assert routes.experts[0].tolist() == [0, 1, 2, 3] and bool(routes.weights.isnan().all())
    x[1] = float("nan")
    routes = experts.route_rows(x, router[:, 4:].contiguous(), 3)
    assert routes.experts[1].tolist() == [0, 1, 2] and bool(routes.weights[1].isnan().all()) and bool(routes.weights[::2].isfinite().all())


def test_no_tokens():
    from fastmace_b200 import experts
    x = torch.zeros(0, 16, device="cuda")
    routes = experts.route_rows(x, torch.zeros(16, 4, device="cuda"), 2)
    assert routes.experts.shape == routes.weights.shape == (0, 2)
    assert experts.expert_layer(x, torch.zeros(4, 16, 8, device="cuda"), torch.zeros(4, 4, 16, device="cuda"), routes).shape == (0, 16)


def test_captured_and_replayed_on_other_tokens():
    from fastmace_b200 import experts, grouped
    g = torch.Generator(device="cuda").manual_seed(6)
    x, up, down = _layer(6, 16, 256, 128, BF16, g)
    router = torch.randn(256, 16, generator=g, device="cuda").to(BF16)

    def run():
        routes = experts.route_rows(x, router, 4)
        return experts.expert_layer(x, up, down, routes)

    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for _ in range(2):                                     # two graphs, whose scratch is their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                y = run()
        graphs.append((graph, y))
    for _ in range(3):
        x.copy_(torch.randn(6, 256, generator=g, device="cuda"))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = run()
        assert all(torch.equal(y, want) for _, y in graphs)
    grouped.check_status()


def test_calls_on_two_streams():
    from fastmace_b200 import experts, grouped
    g = torch.Generator(device="cuda").manual_seed(8)
    layers = [_layer(20, 16, 512, 256, BF16, g) for _ in range(2)]
    routes = experts.Routes(torch.randint(0, 16, (20, 4), generator=g, device="cuda", dtype=torch.int32), torch.rand(20, 4, generator=g, device="cuda"))
    want = [experts.expert_layer(*layer, routes) for layer in layers]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for layer, stream in zip(layers, streams):
            with torch.cuda.stream(stream):
                got.append(experts.expert_layer(*layer, routes))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    grouped.check_status()


def test_refusals():
    from fastmace_b200 import experts as m
    x, up, down = torch.zeros(4, 16, device="cuda"), torch.zeros(3, 16, 8, device="cuda"), torch.zeros(3, 4, 16, device="cuda")
    router = torch.zeros(16, 3, device="cuda")
    routes = m.route_rows(x, router, 2)
    many = torch.zeros(129, 16, device="cuda")
    for call in (lambda: m.route_rows(x, router, 0), lambda: m.route_rows(x, router, 4), lambda: m.route_rows(x, router.to(BF16), 2),
                 lambda: m.route_rows(x, router[:8], 2), lambda: m.route_rows(x.double(), router.double(), 2), lambda: m.route_rows(x[0], router, 2),
                 lambda: m.route_rows(x, torch.zeros(16, 1025, device="cuda"), 2), lambda: m.route_rows(x, torch.zeros(16, 64, device="cuda"), 17),
                 lambda: m.route_rows(x, router.t(), 2), lambda: m.route_rows(x.cpu(), router, 2),
                 lambda: m.expert_layer(x, up, down[:2], routes), lambda: m.expert_layer(x, up[:, :, :7], down, routes),
                 lambda: m.expert_layer(x, up, down[:, :3], routes), lambda: m.expert_layer(x.to(BF16), up, down, routes),
                 lambda: m.expert_layer(x, up.permute(0, 2, 1), down, routes), lambda: m.expert_layer(x[:3], up, down, routes),
                 lambda: m.expert_layer(x, up, down, m.Routes(routes.experts.long(), routes.weights)),
                 lambda: m.expert_layer(x, up, down, m.Routes(routes.experts, routes.weights[:, :1])),
                 lambda: m.expert_layer(x, up, down, m.Routes(routes.experts.t().contiguous().t(), routes.weights)),
                 lambda: m.expert_layer(x, up, down, routes, out=x), lambda: m.expert_layer(x, up, down, routes, out=torch.zeros(3, 16, device="cuda")),
                 lambda: m.expert_layer(x, up, down, routes, out=torch.zeros(4, 16, device="cuda", dtype=BF16)),
                 lambda: m.expert_layer(many, up, down, m.route_rows(many, router, 2)), lambda: m.expert_layer(x, up.cpu(), down, routes)):
        with pytest.raises(ValueError):
            call()
