"""What the expert layer keeps of its numbers.

Between the products h = silu(a) b has 17 bits with bfloat16 weights (two bfloat16, each off by half a step: 2^-9 2^-9 of h) and 23 with the others (two
tf32, of 11 bits with a sign between them: a step of 24 bits). The tests' a are 64, where silu(a) = a in float32, and their b are sums of powers of two that
float32 holds; a column of the second matrix takes one h less another, so y is their difference, off by what the two lose, and rounded once.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens,width,inner,columns", [(1, 8, 2, 8), (9, 40, 70, 64), (17, 264, 1032, 136), (33, 33, 515, 101)])
def test_what_passes_the_gate_keeps_its_bits(tokens, width, inner, columns, dtype):
    from fastmace_b200 import experts
    width = max(width, columns)
    x = torch.zeros(tokens, width, device="cuda")
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -9, 2.0 ** -20
    x *= torch.exp2(torch.arange(tokens, device="cuda") % 3).unsqueeze(1)       # b by token: 1, 2 or 4 times
    up = torch.zeros(1, width, 2 * inner, device="cuda")
    up[:, 0, :inner] = 64.0
    up[:, :2, inner:] = 1.0                                                       # b = 1 + 2^-9, and 2^-20 more in every second column
    up[:, 2, inner::2] = 1.0
    down = torch.zeros(1, inner, width, device="cuda")
    for c in range(columns):
        down[0, 2 * c % (inner - inner % 2), c] = 1.0
        down[0, (2 * c * 7 + 1) % (inner - inner % 2), c] = -1.0
    routes = experts.Routes(torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), torch.ones(tokens, 1, device="cuda"))
    y = experts.expert_layer(x.to(dtype), up.to(dtype), down.to(dtype), routes)[:, :columns].double()
    scale = torch.exp2(torch.arange(tokens, device="cuda") % 3).double().unsqueeze(1)
    h = 64.0 * scale * scale                                                      # (a is 64 times as large as well)
    want = h * 2.0 ** -20
    lost = 2.0 ** -18 if dtype == BF16 else 2.0 ** -23
    assert bool(((y - want).abs() <= 2 * h * 1.01 * lost + torch.finfo(dtype).eps / 2 * want).all()), (float(y.min()), float(y.max()))


def _like(y, ref, off):
    """The same infinities and NaN as the reference; what is finite within `off`, and one rounding."""
    half = torch.finfo(y.dtype).eps / 2
    y = y.double()
    assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y.isinf(), ref.isinf()), (y, ref)
    assert torch.equal(y[ref.isinf()], ref[ref.isinf()])
    fine = ref.isfinite()
    assert bool(((y - ref).abs()[fine] <= (off + half * ref.abs())[fine]).all())


def _plain(x, up, down):
    """The layer with one expert and weights 1 in float64, and how far a sum may be off: (t + 8) 2^-24 of the absolute sums and what
    operands lose, 2^-20; twice, through a slope below 1.1 and factors of at most the largest h."""
    x, up, down = x.double(), up[0].double(), down[0].double()
    a, b = (x @ up).chunk(2, 1)
    h = a / (1 + torch.exp(-a)) * b
    return h @ down, h


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width,inner", [(64, 32), (65, 33), (2056, 24), (40, 1032)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_infinities_give_what_a_plain_product_gives(width, inner, sign, dtype):
    from fastmace_b200 import experts, grouped
    tokens, inf = 12, float("inf")
    g = torch.Generator(device="cuda").manual_seed(width + inner)
    x = torch.randint(-3, 4, (tokens, width), generator=g, device="cuda").to(dtype)
    up = (torch.randint(1, 3, (1, width, 2 * inner), generator=g, device="cuda") * 2.0 ** -8).to(dtype)          # positive: infinities keep their sign
    down = torch.randint(1, 4, (1, inner, width), generator=g, device="cuda").to(dtype)
    down[:, :, 1::2] *= -1
    routes = experts.Routes(torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), torch.ones(tokens, 1, device="cuda"))
    want = experts.expert_layer(x, up, down, routes)
    rest = torch.arange(tokens, device="cuda") != 3
    # an infinite x: both halves of its row are infinite (silu(-inf) is -inf / inf, not a number)
    bad = x.clone()
    bad[3, 5] = sign * inf
    y = experts.expert_layer(bad, up, down, routes)
    assert torch.equal(y[rest], want[rest])
    _like(y[3:4], _plain(bad, up, down)[0][3:4], 0.0)
    assert bool(y[3].isinf().all()) if sign > 0 else bool(y[3].isnan().all())
    # an infinite weight that multiplies the gate: one h of each token is infinite, or not a number where x is zero
    heavy = up.clone()
    heavy[0, 7, inner + inner // 2] = sign * inf
    _like(experts.expert_layer(x, heavy, down, routes), _plain(x, heavy, down)[0], 0.0)
    # an infinite weight of the second matrix: its column alone, by the sign of h
    heavy = down.clone()
    heavy[0, inner - 1, width - 2] = sign * inf
    y, (ref, h) = experts.expert_layer(x, up, heavy, routes), _plain(x, up, heavy)
    others = torch.arange(width, device="cuda") != width - 2
    assert torch.equal(y[:, others], want[:, others])
    clear = h[:, inner - 1].abs() > 1e-9          # (an h that is zero but for roundings has no sign)
    _like(y[clear, width - 2], ref[clear, width - 2], 0.0)
    assert bool(y[clear, width - 2].isinf().all())
    # two that cancel
    heavy[0, 0, width - 2] = -sign * inf
    y, (ref, h) = experts.expert_layer(x, up, heavy, routes), _plain(x, up, heavy)
    clear &= h[:, 0].abs() > 1e-9
    _like(y[clear, width - 2], ref[clear, width - 2], 0.0)
    grouped.check_status()


def test_numbers_near_the_largest_stay_finite():
    """Parts of operands: what is rounded to them may not become infinite."""
    from fastmace_b200 import experts
    largest = torch.finfo(F32).max
    one = lambda dtype: experts.Routes(torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda"))  # noqa: E731

    def layer(dtype, x, a, b, w):
        """y of one token whose first x alone is not zero, one inner column and weights a, b, w."""
        rows, up, down = (torch.zeros(shape, dtype=dtype, device="cuda") for shape in ((1, 16), (1, 16, 16), (1, 8, 16)))
        rows[0, 0], up[0, 0, 0], up[0, 0, 8], down[0, 0] = x, a, b, w
        return experts.expert_layer(rows, up, down, one(dtype))[0].double()

    small = 2.0 ** -120
    cases = [(F32, small, largest, 1.0 / small, 1.0), (F32, largest, 16 * small, small, 1.0 / 32), (F32, small, 64.0 / small, 2.0 ** -16 / small, -largest),
             (F32, 64.0, 1.0, largest * 0.9999 / 4096, 2.0 ** -20), (F32, 1.0, 64.0, largest * 0.9999 / 64, 2.0 ** -20)]
    for x in range(64, 128):                      # an h beyond bfloat16's largest number
        b = float(torch.tensor(largest * 0.9992 / x ** 2, dtype=BF16))
        if 0.9985 < x ** 2 * b / largest < 0.9999:
            cases.append((BF16, float(x), 1.0, b, 2.0 ** -20))
    assert len(cases) > 5
    for dtype, x, a, b, w in cases:
        held = [float(torch.tensor(v, dtype=dtype)) for v in (x, a, b, w)]
        gate = held[0] * held[1]
        want = gate / (1 + float(torch.exp(torch.tensor(-gate, dtype=torch.float64)))) * (held[0] * held[2]) * held[3]
        y = layer(dtype, *held)
        assert bool(((y - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -17) * abs(want)).all()), (dtype, x, a, b, w, float(y[0]), want)


@pytest.mark.parametrize("tokens,experts,top,width,inner", [(17, 12, 4, 4096, 128), (5, 3, 2, 1024, 4100), (8, 4, 2, 4096, 4096), (33, 9, 3, 515, 1001),
                                                            (64, 4, 2, 512, 256), (1, 64, 8, 2048, 1024)])
def test_float32_layers_are_as_near_as_float32_is(tokens, experts, top, width, inner):
    """Each product's terms are off by 2^-21 of themselves at most (two operands by 2^-23 each, the product of their rests, 2^-22, left out), in either
    direction alike, and so is their sum, of terms of either sign, on the norm; roundings of a sum in stages are less. Two products behind one
    another, whose errors are independent: 2^-20.5."""
    from fastmace_b200 import experts as m
    g = torch.Generator(device="cuda").manual_seed(width + inner)
    x = torch.randn(tokens, width, generator=g, device="cuda")
    up = torch.randn(experts, width, 2 * inner, generator=g, device="cuda") / width ** 0.5
    down = torch.randn(experts, inner, width, generator=g, device="cuda") / inner ** 0.5
    chosen = torch.stack([torch.randperm(experts, generator=g, device="cuda")[:top] for _ in range(tokens)]).to(torch.int32)
    weights = torch.rand(tokens, top, generator=g, device="cuda")
    y = m.expert_layer(x, up, down, m.Routes(chosen, weights)).double()
    ref = torch.zeros_like(y)
    for e in range(experts):
        t, j = torch.nonzero(chosen == e, as_tuple=True)
        a, b = (x[t].double() @ up[e].double()).chunk(2, 1)
        ref.index_add_(0, t, (a / (1 + torch.exp(-a)) * b) @ down[e].double() * weights[t, j].double()[:, None])
    assert float((y - ref).norm() / ref.norm()) < 2.0 ** -20.5


@pytest.mark.parametrize("small", ["x", "up", "down"])
def test_float32_layers_at_the_end_of_their_range(small):
    """A tf32's smallest step is 2^-136, which an operand loses at most beside what operands of any size do; from 2^-112 on that is no more than the last
    of its 24 bits. Weights here are smaller, by the root of the depth: 2^-116 and 2^-115.5 of the norm, so that the step is 2^-20 and 2^-20.5 of
    them, and as much of their sums' norm, added to the 2^-20.5 of two products."""
    from fastmace_b200 import experts
    tokens, width, inner, scale = 9, 264, 136, 2.0 ** -112
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(tokens, width, generator=g, device="cuda")
    up = torch.randn(1, width, 2 * inner, generator=g, device="cuda") / width ** 0.5
    down = torch.randn(1, inner, width, generator=g, device="cuda") / inner ** 0.5
    if small == "x":
        x, up = x * scale, up / scale
    elif small == "up":
        x, up = x / scale, up * scale
    else:
        up[:, :, inner:] /= scale
        down *= scale
    y = experts.expert_layer(x, up, down, experts.Routes(torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), torch.ones(tokens, 1, device="cuda")))
    ref, _ = _plain(x, up, down)
    operand = {"x": x, "up": up[:, :, :inner], "down": down}[small].double()
    step = 2.0 ** -136 / float(operand.square().mean().sqrt())
    assert float((y.double() - ref).norm() / ref.norm()) < 2.0 ** -20.5 + step
