"""What the expert layer keeps of its numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


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
