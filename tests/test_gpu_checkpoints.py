"""Rows held in 8 bits, the gate and the backward pass from them, on the GPU against plain float64 evaluations.

Tolerances. Codes and exponents are whole numbers of a definition without rounding before the code's own: they are equal. A held value is
off by half a step of its code: 2^-4 of itself, or half of the smallest code, 2^-10 units. A gate is a product of float32 roundings: the
sigmoid is 1 / (1 + exp(-a)), whose exponential is off by 2 ulp of float32 in float32 results and, in the fast form, by 2 ulp and by the
rounding of a log2(e), |a| 2^-24 of the result: s is off by (|a| + 6) 2^-23 of itself at most. Five products and a sum follow, 2^-24 each of
their own size. Results of 16 bits are rounded once more, eps / 2. The weight gradient: as for rows that are not held, (t + 8) 2^-24 of the
terms' absolute sum.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LIMITS = {F32: (-117, 120), BF16: (-117, 120), F16: (-15, 8)}


def _wide(t, stride):
    if stride == 1:
        return t
    out = torch.full((t.shape[0], stride, t.shape[1]), float("nan"), dtype=t.dtype, device=t.device)
    out[:, 0] = t
    return out[:, 0]


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)


def _hold(x, dtype):
    """(values held, exponents) by the definition: the smallest unit that holds the block, and the nearest code, ties to even."""
    low, high = LIMITS[dtype]
    b = _blocks(x.double())
    finite = torch.where(b.isfinite(), b, 0.0).abs().amax(2)
    e = torch.full_like(finite, low)
    for k in range(low, high):
        e = torch.where(finite > 448 * 2.0 ** k, float(k + 1), e)
    unit = torch.exp2(e)[:, :, None]
    v = b / unit
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    most = torch.where(e == high, 240.0, 448.0)[:, :, None]
    code = torch.minimum(torch.maximum(torch.round(v / step) * step, -most), most)
    code = torch.where(b.isfinite(), code, float("nan"))
    return (code * unit).reshape(x.shape[0], -1)[:, :x.shape[1]], (e + 127).to(torch.uint8)


def _rows(rows, columns, dtype, g):
    """Values of very different sizes, some zeros, a row of zeros, a block at each end of the type's range."""
    x = torch.randn(rows, columns, generator=g, device="cuda") * torch.exp(3 * torch.randn(rows, 1, generator=g, device="cuda"))
    x = x * torch.exp(2 * torch.randn(columns, generator=g, device="cuda"))
    x = torch.where(torch.rand(rows, columns, generator=g, device="cuda") < 0.1, 0.0, x).clamp(-6e4, 6e4).to(dtype)
    info = torch.finfo(dtype)
    for row, value in enumerate((0.0, info.max, info.tiny, info.tiny / 4, 448.0, 449.0, 0.875 * info.max)):
        if row + 1 < rows:
            x[row] = torch.where(torch.rand(columns, generator=g, device="cuda") < 0.5, -value, value).to(dtype)
    return x


SHAPES = [(1, 1, 1), (1, 32, 1), (3, 31, 1), (9, 33, 2), (40, 64, 3), (33, 8, 1), (17, 515, 1), (50, 1000, 2), (300, 2048, 1), (10, 2049, 1),
          (2, 5000, 1), (5000, 40, 1), (3, 16384, 1)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_held_rows_are_the_nearest_codes(shape, dtype):
    from fastmace_b200 import checkpoints
    rows, columns, stride = shape
    g = torch.Generator(device="cuda").manual_seed(rows + columns)
    x = _rows(rows, columns, dtype, g)
    for parts in (1, 2) if columns % 2 == 0 else (1,):
        held = checkpoints.hold_rows(_wide(x, stride), parts)
        want = [_hold(h, dtype) for h in x.chunk(parts, 1)]
        values, exponents = (torch.cat(t, 1) for t in zip(*want))
        back = checkpoints.release_rows(held)
        assert torch.equal(held.exponents, exponents)
        assert back.dtype == dtype and torch.equal(back.double(), values) and bool(back.isfinite().all())
        # (off by half a code; in the highest unit, whose codes end at 240, by a sixteenth too)
        unit = torch.exp2(exponents.double() - 127).view(rows, parts, -1).repeat_interleave(32, 2)[:, :, :columns // parts].reshape(rows, columns)
        assert bool(((back.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * unit).all())
        given = torch.full((rows, 3, columns), 7.0, device="cuda", dtype=dtype)
        checkpoints.release_rows(held, out=given[:, 1])
        assert torch.equal(given[:, 1], back) and bool((given[:, 0] == 7).all()) and bool((given[:, 2] == 7).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_what_is_not_finite_is_nan_and_leaves_its_block(dtype):
    from fastmace_b200 import checkpoints
    for columns in (64, 33):
        x = torch.full((4, columns), 3.0, device="cuda", dtype=dtype)
        x[0, 1], x[1, 2], x[2, 30] = float("inf"), float("-inf"), float("nan")
        x[3] = float("nan")
        back = checkpoints.release_rows(checkpoints.hold_rows(x))
        assert torch.equal(back.isnan(), ~x.isfinite()) and bool((back[x.isfinite()] == 3).all())


def _gate(u):
    a, b = u.double().chunk(2, 1)
    s = 1 / (1 + torch.exp(-a))
    return a, b, s


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1, 2, 1), (5, 66, 1), (33, 128, 2), (40, 1030, 1), (100, 2048, 1), (3, 16, 1), (7, 8192, 1), (3000, 48, 4)])
def test_gate_and_its_gradient_against_float64(shape, dtype):
    from fastmace_b200 import checkpoints
    rows, columns, stride = shape
    g = torch.Generator(device="cuda").manual_seed(columns)
    u = (torch.randn(rows, columns, generator=g, device="cuda") * 4).to(dtype)
    dh = torch.randn(rows, columns // 2, generator=g, device="cuda").to(dtype)
    half, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == F16 else 0.0
    h, held = checkpoints.gated_rows(_wide(u, stride), hold=True)
    assert torch.equal(h, checkpoints.gated_rows(u))
    want = checkpoints.hold_rows(u, parts=2)
    assert held.parts == 2 and torch.equal(held.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(held.exponents, want.exponents)

    def near(x, ref, size):
        assert x.dtype == dtype and bool(((x.double() - ref).abs() <= size + half * (ref.abs() + size) + tiny).all())

    back = checkpoints.release_rows(held)
    for source, rows_of in ((held, back), (u, u), (_wide(u, stride), u)):
        a, b, s = _gate(rows_of)
        off = (a.abs() + 6) * 2.0 ** -23                  # of s, relative
        du, anew = checkpoints.gated_rows_gradient(source, _wide(dh, stride))
        near(anew, a * s * b, (a * s * b).abs() * (off + 2.0 ** -22))
        d = dh.double()
        slope = s.abs() * (1 + a.abs() * (1 - s).abs())
        # 1 - s is off by s off and by its own rounding, 2^-24
        parts = (d * b).abs() * (slope * (off + 2.0 ** -21) + s * a.abs() * (s * off + 2.0 ** -23))
        near(du[:, :columns // 2], d * b * s * (1 + a * (1 - s)), parts)
        near(du[:, columns // 2:], d * a * s, (d * a * s).abs() * (off + 2.0 ** -22))
        again, none = checkpoints.gated_rows_gradient(source, dh, recompute=False)
        assert none is None and torch.equal(again, du)
    a, b, s = _gate(u)
    near(h, a * s * b, (a * s * b).abs() * ((a.abs() + 6) * 2.0 ** -23 + 2.0 ** -22))


def test_gate_gradient_against_differences():
    from fastmace_b200 import checkpoints
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.randn(20, 64, generator=g, device="cuda")
    dh, step = torch.randn(20, 32, generator=g, device="cuda"), torch.randn(20, 64, generator=g, device="cuda")
    loss = lambda x: float((checkpoints.gated_rows(x).double() * dh.double()).sum())  # noqa: E731
    du, _ = checkpoints.gated_rows_gradient(u, dh)
    t = 2.0 ** -8
    slope = (loss(u + t * step) - loss(u - t * step)) / (2 * t)
    # the third derivative times t^2 / 6 and roundings of 640 terms over 2 t
    assert abs(slope - float((du.double() * step.double()).sum())) < 2e-2


def test_gate_far_from_zero():
    from fastmace_b200 import checkpoints
    for dtype in (F32, BF16):
        a = torch.tensor([-200.0, -90.0, -87.0, 90.0, 200.0, 0.0], device="cuda", dtype=dtype)
        u = torch.cat([a, torch.ones_like(a)])[None]
        h = checkpoints.gated_rows(u)
        assert bool(h.isfinite().all()) and h[0, 3:].tolist() == a[3:].tolist() and bool((h[0, :3].abs() < 1e-30).all())
        du, _ = checkpoints.gated_rows_gradient(u, torch.ones(1, 6, device="cuda", dtype=dtype))
        assert bool(du.isfinite().all()) and du[0, 4] == 1 and du[0, 5] == 0.5


# rows, groups, k, n, share of rows without a group
PRODUCTS = [(1, 1, 1, 1, 0.0), (7, 3, 33, 20, 0.0), (200, 5, 128, 128, 0.1), (257, 3, 65, 129, 0.0), (1000, 7, 130, 515, 0.3), (300, 6, 96, 64, 1.0),
            (2500, 3, 1024, 256, 0.0), (5000, 8, 128, 128, 0.0), (9000, 30, 520, 264, 0.1), (6000, 5, 1032, 1040, 0.0), (20_000, 7, 200, 1096, 0.0)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", PRODUCTS)
def test_weight_gradient_of_held_rows(shape, dtype):
    from fastmace_b200 import checkpoints, grouped
    rows, groups, k, n, absent = shape
    g = torch.Generator(device="cuda").manual_seed(rows + k)
    keys = torch.randint(0, groups, (rows,), generator=g, device="cuda", dtype=torch.int32)
    keys = torch.where(torch.rand(rows, generator=g, device="cuda") < absent, -1, keys).to(torch.int32)
    plan = grouped.group_rows(keys, groups)
    x = (torch.randn(rows, k, generator=g, device="cuda") * torch.exp(torch.randn(k, generator=g, device="cuda"))).to(dtype)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    held = checkpoints.hold_rows(x)
    back = checkpoints.release_rows(held)
    dw = checkpoints.held_weight_gradient(held, dy, plan)
    for q in range(groups):
        r = (keys == q).nonzero()[:, 0]
        a, b = back[r].double(), dy[r].double()
        assert bool(((dw[q].double() - a.t() @ b).abs() <= (len(r) + 8) * 2.0 ** -24 * (a.abs().t() @ b.abs())).all()), (q, len(r))
    # the bits of the product with rows that have been read back, and of the same call again
    if k % 8 == 0:
        assert torch.equal(dw, grouped.grouped_linear_weight_gradient(back, dy, plan))
    assert torch.equal(dw, checkpoints.held_weight_gradient(held, dy, plan))
    more = torch.ones_like(dw)
    checkpoints.held_weight_gradient(held, dy, plan, out=more, accumulate=True)
    assert bool(((more - 1 - dw).abs() <= 2.0 ** -22 * (dw.abs() + 1)).all())
    grouped.check_status()


def test_no_rows():
    from fastmace_b200 import checkpoints, grouped
    x = torch.zeros(0, 64, device="cuda")
    held = checkpoints.hold_rows(x, parts=2)
    assert checkpoints.release_rows(held).shape == (0, 64)
    h, again = checkpoints.gated_rows(x, hold=True)
    du, anew = checkpoints.gated_rows_gradient(again, torch.zeros(0, 32, device="cuda"))
    assert h.shape == anew.shape == (0, 32) and du.shape == (0, 64)
    plan = grouped.group_rows(torch.zeros(0, dtype=torch.int32, device="cuda"), 3)
    assert bool((checkpoints.held_weight_gradient(checkpoints.hold_rows(x), torch.zeros(0, 8, device="cuda"), plan) == 0).all())


def test_captured_and_replayed_on_other_rows():
    from fastmace_b200 import checkpoints, grouped
    g = torch.Generator(device="cuda").manual_seed(5)
    u, dh, dy = (torch.randn(700, c, generator=g, device="cuda").to(BF16) for c in (256, 128, 64))
    plan = grouped.group_rows(torch.randint(0, 4, (700,), generator=g, device="cuda"), 4)

    def run():
        h, held = checkpoints.gated_rows(u, hold=True)
        du, anew = checkpoints.gated_rows_gradient(held, dh)
        return h, du, anew, checkpoints.held_weight_gradient(checkpoints.hold_rows(h), dy, plan)

    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = run()
    for _ in range(2):
        u.copy_(torch.randn(700, 256, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run()))


def test_refusals():
    from fastmace_b200 import checkpoints as c
    from fastmace_b200 import grouped
    x = torch.zeros(4, 64, device="cuda", dtype=BF16)
    held, two = c.hold_rows(x), c.hold_rows(x, parts=2)
    dh, dy = torch.zeros(4, 32, device="cuda", dtype=BF16), torch.zeros(4, 8, device="cuda", dtype=BF16)
    plan = grouped.group_rows(torch.zeros(4, dtype=torch.int32, device="cuda"), 2)
    for call in (lambda: c.hold_rows(x.double()), lambda: c.hold_rows(x[0]), lambda: c.hold_rows(x, parts=3), lambda: c.hold_rows(x[:, :63], parts=2),
                 lambda: c.hold_rows(x.t()), lambda: c.release_rows(held._replace(codes=held.codes.view(torch.uint8))),
                 lambda: c.release_rows(held._replace(exponents=held.exponents[:, :1])), lambda: c.release_rows(held._replace(parts=4)),
                 lambda: c.release_rows(held._replace(dtype=torch.float64)), lambda: c.release_rows(held, out=torch.zeros(4, 64, device="cuda")),
                 lambda: c.release_rows(held._replace(codes=held.codes[:, :32], exponents=held.exponents[:, :1])),
                 lambda: c.gated_rows(x[:, :63]), lambda: c.gated_rows(x, out=x[:, :32]), lambda: c.gated_rows(x, out=dh.float()),
                 lambda: c.gated_rows_gradient(held, dh), lambda: c.gated_rows_gradient(two, dh.float()), lambda: c.gated_rows_gradient(two, x),
                 lambda: c.gated_rows_gradient(x, dh, out=x), lambda: c.gated_rows_gradient(two, dh[:3]),
                 lambda: c.held_weight_gradient(two, dy, plan), lambda: c.held_weight_gradient(held, dy.float(), plan),
                 lambda: c.held_weight_gradient(held, dy[:3], plan), lambda: c.held_weight_gradient(held, dy, plan, accumulate=True),
                 lambda: c.held_weight_gradient(held._replace(codes=held.codes.cpu()), dy, plan)):
        with pytest.raises(ValueError):
            call()
