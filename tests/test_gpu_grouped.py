"""Grouped products and their gradients on the GPU against plain float64 matrix products, group by group.

Tolerances, per element, with S = sum of |x| |w| over the terms of the sum: a float32 sum of t terms in any order, with
rounded or truncated additions, is off by at most about t 2^-24 S to t 2^-23 S in the worst case; the kernels add 16 products at a time and
restart their accumulators, which leaves far fewer additions in a chain than terms, so (t + 8) 2^-24 S bounds them. Products
of 16-bit numbers are exact in float32. A 16-bit output is rounded once more: half a step, eps / 2 of the value, and half the
smallest subnormal (float16: 2^-25).
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _keys(rows, groups, kind, rng):
    if kind == "even":
        keys = rng.integers(0, groups, rows)
    elif kind == "one":                                    # every row in the last group, the others empty
        keys = np.full(rows, groups - 1)
    elif kind == "none":
        keys = np.full(rows, -1)
    else:                                                  # uneven, with rows of no group on both sides of the range
        keys = np.minimum((rng.pareto(1.0, rows) * 2).astype(np.int64), groups + 2) - 1
    return torch.tensor(keys, dtype=torch.int32, device="cuda")


def _wide(t, stride):
    """The same matrix as a view with rows `stride` times as far apart; NaN in between."""
    if stride == 1:
        return t
    out = torch.full((t.shape[0], stride, t.shape[1]), float("nan"), dtype=t.dtype, device=t.device)
    out[:, 0] = t
    return out[:, 0]


def _rounding(t):
    return 0.0 if t == F32 else torch.finfo(t).eps / 2


def _smallest(t):
    return 2.0 ** -25 if t == F16 else 0.0


def _check_rows(y, x, w, keys, transposed=False):
    groups = w.shape[0]
    ref = torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(ref)
    for g in range(groups):
        r = (keys == g).nonzero()[:, 0]
        if len(r):
            a, b = x[r].double(), w[g].double()
            b = b.t() if transposed else b
            ref[r], size[r] = a @ b, a.abs() @ b.abs()
    terms = x.shape[1]
    tol = (terms + 8) * 2.0 ** -24 * size
    tol = tol + _rounding(y.dtype) * (ref.abs() + tol) + _smallest(y.dtype)
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), f"largest excess {float((off - tol).max())}, rel {float(off.norm() / ref.norm())}"


def _check_weights(dw, x, dy, keys, base=None):
    for g in range(dw.shape[0]):
        r = (keys == g).nonzero()[:, 0]
        a, b = x[r].double(), dy[r].double()
        ref, size = a.t() @ b, a.abs().t() @ b.abs()
        if base is not None:
            ref, size = ref + base[g].double(), size + base[g].abs().double()
        off = (dw[g].double() - ref).abs()
        assert bool((off <= (len(r) + 8) * 2.0 ** -24 * size).all()), (g, len(r), float(off.max()))
        if not len(r) and base is None:
            assert bool((dw[g] == 0).all())


# rows, groups, k, n, spread of the keys, row stride
SHAPES = [(1, 1, 1, 1, "even", 1), (1, 3, 128, 128, "one", 1), (7, 64, 64, 32, "even", 1), (33, 2, 16, 8, "uneven", 1),
          (200, 5, 128, 128, "even", 4), (257, 3, 65, 129, "uneven", 1), (100, 9, 1, 200, "even", 1), (90, 4, 200, 1, "even", 3),
          (513, 17, 100, 72, "uneven", 1), (1000, 7, 130, 515, "even", 1), (640, 2, 264, 384, "one", 2),
          (300, 6, 128, 64, "none", 1), (5000, 8, 128, 128, "uneven", 4), (129, 1024, 48, 56, "even", 1),
          (20_000, 7, 200, 1096, "uneven", 1), (9000, 30, 520, 264, "even", 1), (6000, 5, 1032, 1040, "uneven", 2), (2500, 3, 1024, 256, "even", 1), (700, 2, 2056, 136, "uneven", 1), (16, 4, 4096, 512, "even", 1)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_products_and_gradients_against_float64(shape, dtype):
    from fastmace_b200 import grouped
    rows, groups, k, n, spread, stride = shape
    rng = np.random.default_rng(rows + 7 * n)
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    keys = _keys(rows, groups, spread, rng)
    plan = grouped.group_rows(keys, groups)
    x = _wide(torch.randn(rows, k, generator=g, device="cuda").to(dtype), stride)
    dy = _wide(torch.randn(rows, n, generator=g, device="cuda").to(dtype), stride)
    w = (torch.randn(groups, k, n, generator=g, device="cuda") / k ** 0.5).to(dtype)
    y = grouped.grouped_linear(x, w, plan)
    dx = grouped.grouped_linear_input_gradient(dy, w, plan)
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan)
    assert y.dtype == dx.dtype == dtype and dw.dtype == F32
    _check_rows(y, x, w, keys)
    _check_rows(dx, dy, w, keys, transposed=True)
    _check_weights(dw, x, dy, keys)
    # the same bits again
    assert torch.equal(y, grouped.grouped_linear(x, w, plan))
    assert torch.equal(dx, grouped.grouped_linear_input_gradient(dy, w, plan))
    assert torch.equal(dw, grouped.grouped_linear_weight_gradient(x, dy, plan))
    grouped.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(40_000, 3, 128, 128, "uneven", 4), (30_000, 2, 72, 40, "even", 1), (20_000, 40, 136, 264, "uneven", 1)])
def test_long_groups_against_float64(shape, dtype):
    from fastmace_b200 import grouped
    rows, groups, k, n, spread, stride = shape
    rng = np.random.default_rng(3)
    g = torch.Generator(device="cuda").manual_seed(11)
    keys = _keys(rows, groups, spread, rng)
    plan = grouped.group_rows(keys, groups)
    # positive values: every addition of a sum loses in the same direction
    x = _wide(torch.rand(rows, k, generator=g, device="cuda").to(dtype), stride)
    dy = torch.rand(rows, n, generator=g, device="cuda").to(dtype)
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan)
    _check_weights(dw, x, dy, keys)
    w = torch.rand(groups, k, n, generator=g, device="cuda").to(dtype)
    _check_rows(grouped.grouped_linear(x, w, plan), x, w, keys)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("groups,k,n", [(310, 100, 60), (170, 130, 190), (60, 264, 600), (1024, 8, 3)])
def test_weight_gradient_of_a_long_group_among_short_ones(groups, k, n, dtype):
    """Many groups, of which one has two rows in three and another a fifth: these are cut, the others are not."""
    from fastmace_b200 import grouped
    rows = 24_001
    rng = np.random.default_rng(groups)
    keys = rng.integers(-1, groups, rows)
    draw = rng.random(rows)
    keys[draw < 0.66], keys[draw > 0.8] = groups // 2, groups - 1
    keys = torch.tensor(keys, dtype=torch.int32, device="cuda")
    plan = grouped.group_rows(keys, groups)
    g = torch.Generator(device="cuda").manual_seed(groups)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan)
    _check_weights(dw, x, dy, keys)
    base = torch.randn(groups, k, n, generator=g, device="cuda")
    added = grouped.grouped_linear_weight_gradient(x, dy, plan, out=base.clone(), accumulate=True)
    _check_weights(added, x, dy, keys, base)
    assert torch.equal(dw, grouped.grouped_linear_weight_gradient(x, dy, plan))
    grouped.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,groups,k,n", [(1, 1, 4096, 40), (1, 64, 2056, 1024), (2, 2, 512, 512), (8, 64, 2048, 1024), (9, 70, 1100, 515),
                                             (30, 1, 515, 300), (31, 2, 640, 96), (5, 1024, 1096, 200), (40, 1, 2100, 136), (70, 3, 2048, 128)])
def test_single_tokens(rows, groups, k, n, dtype):
    """Few rows of deep products, where several blocks share the depth of a tile; some rows belong to no group."""
    from fastmace_b200 import grouped
    rng = np.random.default_rng(rows + k)
    keys = rng.integers(0, groups, rows)
    keys[rng.random(rows) < 0.15] = -1
    keys = torch.tensor(keys, device="cuda")
    plan = grouped.group_rows(keys, groups)
    g = torch.Generator(device="cuda").manual_seed(k)
    w = (torch.randn(groups, k, n, generator=g, device="cuda") / k ** 0.5).to(dtype)
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    y = grouped.grouped_linear(x, w, plan)
    dx = grouped.grouped_linear_input_gradient(dy, w, plan)
    _check_rows(y, x, w, keys)
    _check_rows(dx, dy, w, keys, transposed=True)
    # captured, with other values and other groups at each replay
    slots, inputs = torch.full_like(keys, groups - 1), torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        later = grouped.grouped_linear(inputs, w, grouped.group_rows(slots, groups))
    for shift in range(3):
        slots.copy_((keys + shift) % groups)
        inputs.copy_(x * (shift + 1))
        graph.replay()
        _check_rows(later, inputs, w, slots)
    assert torch.equal(y, grouped.grouped_linear(x, w, plan))
    grouped.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_order_of_magnitude_extremes(dtype):
    """Values from 2^-60 to 2^60 of one matrix: float32 operands keep their 24 bits at every size."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(1)
    keys = torch.arange(300, device="cuda") % 2
    plan = grouped.group_rows(keys, 2)
    size = torch.exp2(torch.randint(-60, 61, (300, 1), generator=g, device="cuda").float())
    x = (torch.randn(300, 128, generator=g, device="cuda") * size).to(dtype)
    w = torch.randn(2, 128, 128, generator=g, device="cuda").to(dtype)
    _check_rows(grouped.grouped_linear(x, w, plan), x, w, keys)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("size", [(64, 128), (65, 129)])
def test_what_is_not_finite_stays_in_its_row_and_group(size, dtype):
    from fastmace_b200 import grouped
    k, n = size
    g = torch.Generator(device="cuda").manual_seed(2)
    keys = torch.tensor([0] * 37 + [1] * 50 + [-1] * 5 + [2] * 40, dtype=torch.int32, device="cuda")
    rows = len(keys)
    plan = grouped.group_rows(keys, 4)                       # group 3 has no rows
    x = torch.randn(rows, k, generator=g, device="cuda").to(dtype)
    dy = torch.randn(rows, n, generator=g, device="cuda").to(dtype)
    w = (torch.randn(4, k, n, generator=g, device="cuda") / 8).to(dtype)
    clean_x, clean_dy, clean_w = x.clone(), dy.clone(), w.clone()
    w[3] = float("nan")
    x[87:92] = float("nan")                                  # rows of no group
    dy[87:92] = float("inf")
    x[40, 3] = float("inf")
    x[41, 5] = float("nan")
    y = grouped.grouped_linear(x, w, plan)
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[40:42] = False
    fine[87:92] = False
    _check_rows(y[fine], clean_x[fine], clean_w, keys[fine])
    assert bool((~torch.isfinite(y[40])).all()) and bool(torch.isnan(y[41]).all()) and bool((y[87:92] == 0).all())
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan)
    assert bool(torch.isfinite(dw[[0, 2, 3]]).all()) and bool((~torch.isfinite(dw[1, [3, 5]])).all())
    keep = keys != 1
    _check_weights(dw[[0, 2, 3]], clean_x[keep], clean_dy[keep], torch.tensor([0] * 37 + [-1] * 5 + [1] * 40, device="cuda"))


def test_given_outputs_keep_the_rows_of_no_group():
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(4)
    keys = torch.tensor(([0, 5, -1, 1] * 30)[:118], dtype=torch.int64, device="cuda")
    plan = grouped.group_rows(keys, 2)
    for dtype, k, n in ((F32, 128, 128), (BF16, 128, 256), (F16, 33, 47)):
        x = torch.randn(118, k, generator=g, device="cuda").to(dtype)
        w = torch.randn(2, k, n, generator=g, device="cuda").to(dtype)
        wide = torch.full((118, 3, n), 7.0, dtype=dtype, device="cuda")
        out = grouped.grouped_linear(x, w, plan, out=wide[:, 1])
        assert out.data_ptr() == wide[:, 1].data_ptr()
        gone = (keys < 0) | (keys > 1)
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 2] == 7).all()) and bool((out[gone] == 7).all())
        _check_rows(out[~gone], x[~gone], w, keys[~gone])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_weights_in_the_layout_of_the_models_dictionary(dtype):
    """``l1.skip.0`` is [channels in, element, channels out]: its permuted view is the call's weight, and the gradient goes to
    the same layout and adds up."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(5)
    raw = torch.randn(128, 11, 128, generator=g, device="cuda").to(dtype)
    keys = torch.randint(0, 11, (700,), generator=g, device="cuda", dtype=torch.int32)
    plan = grouped.group_rows(keys, 11)
    x = torch.randn(700, 4, 128, generator=g, device="cuda").to(dtype)[:, 0]
    dy = torch.randn(700, 128, generator=g, device="cuda").to(dtype)
    w = raw.permute(1, 0, 2)
    _check_rows(grouped.grouped_linear(x, w, plan), x, w, keys)
    _check_rows(grouped.grouped_linear_input_gradient(dy, w, plan), dy, w, keys, transposed=True)
    raw_gradient = torch.full((128, 11, 128), 0.5, device="cuda")
    base = raw_gradient.clone().permute(1, 0, 2)
    grouped.grouped_linear_weight_gradient(x, dy, plan, out=raw_gradient.permute(1, 0, 2), accumulate=True)
    _check_weights(raw_gradient.permute(1, 0, 2), x, dy, keys, base=base)
    grouped.grouped_linear_weight_gradient(x, dy, plan, out=raw_gradient.permute(1, 0, 2))
    _check_weights(raw_gradient.permute(1, 0, 2), x, dy, keys)


def test_gradients_against_differences():
    """sum(c * linear(x, W)) along random directions of x and W: products are linear in either, so a difference over any step is
    the derivative up to rounding. Each sum below has 300 * 40 terms of order 1 that were themselves rounded at 2^-24: 1e-4 of
    the norm of the terms is far above that and far below any wrong gradient."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(6)
    keys = torch.randint(-1, 5, (300,), generator=g, device="cuda", dtype=torch.int32)
    plan = grouped.group_rows(keys, 5)
    x, dx = (torch.randn(300, 52, generator=g, device="cuda") for _ in range(2))
    w, dw = (torch.randn(5, 52, 40, generator=g, device="cuda") for _ in range(2))
    c = torch.randn(300, 40, generator=g, device="cuda")

    def f(x, w):
        return grouped.grouped_linear(x, w, plan).double()

    size = float((c.double() * f(x, w)).norm())
    along_x = float((c.double() * (f(x + 0.5 * dx, w) - f(x - 0.5 * dx, w))).sum())
    along_w = float((c.double() * (f(x, w + 0.5 * dw) - f(x, w - 0.5 * dw))).sum())
    by_x = float((grouped.grouped_linear_input_gradient(c, w, plan).double() * dx.double()).sum())
    by_w = float((grouped.grouped_linear_weight_gradient(x, c, plan).double() * dw.double()).sum())
    assert abs(along_x - by_x) < 1e-4 * size and abs(along_w - by_w) < 1e-4 * size


@pytest.mark.parametrize("key_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows,groups", [(0, 1), (1, 1), (31, 3), (1000, 1024), (8192, 7), (8193, 7), (8193, 1024), (100_003, 129), (1_000_000, 2)])
def test_rows_by_group(rows, groups, key_type):
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(rows + groups)
    keys = torch.randint(-2, groups + 3, (rows,), generator=g, device="cuda", dtype=torch.int64)
    if key_type == torch.int64 and rows > 4:
        keys[3], keys[4] = 1 << 40, -(1 << 40)
    plan = grouped.group_rows(keys.to(key_type), groups)
    key = torch.where((keys < 0) | (keys >= groups), torch.full_like(keys, groups), keys)
    assert torch.equal(plan.rows.long(), torch.sort(key, stable=True).indices)
    starts = torch.cat([key.new_zeros(1), torch.bincount(key, minlength=groups + 1)[:groups].cumsum(0)])
    assert torch.equal(plan.offsets.long(), starts)


def test_no_rows():
    from fastmace_b200 import grouped
    plan = grouped.group_rows(torch.zeros(0, dtype=torch.int32, device="cuda"), 3)
    x, w = torch.zeros(0, 16, device="cuda"), torch.ones(3, 16, 8, device="cuda")
    assert grouped.grouped_linear(x, w, plan).shape == (0, 8)
    dw = grouped.grouped_linear_weight_gradient(x, torch.zeros(0, 8, device="cuda"), plan)
    assert dw.shape == (3, 16, 8) and bool((dw == 0).all())
    kept = torch.ones(3, 16, 8, device="cuda")
    grouped.grouped_linear_weight_gradient(x, torch.zeros(0, 8, device="cuda"), plan, out=kept, accumulate=True)
    assert bool((kept == 1).all())


def test_row_numbers_out_of_range_are_skipped():
    """Order and offsets that no group_rows wrote: what is out of range is not read or written."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(8)
    for dtype, k, n in ((F32, 64, 64), (BF16, 64, 128), (BF16, 35, 21)):
        x = torch.randn(64, k, generator=g, device="cuda").to(dtype)
        dy = torch.randn(64, n, generator=g, device="cuda").to(dtype)
        w = torch.randn(2, k, n, generator=g, device="cuda").to(dtype)
        order = torch.arange(64, dtype=torch.int32, device="cuda")
        order[5], order[40] = 64, -3
        bad = grouped.RowGroups(order, torch.tensor([0, 32, 900], dtype=torch.int32, device="cuda"))
        keys = torch.tensor([0] * 32 + [1] * 32, device="cuda")
        keys[5] = keys[40] = -1
        out = torch.zeros(64, n, dtype=dtype, device="cuda")
        _check_rows(grouped.grouped_linear(x, w, bad, out=out), x, w, keys)
        _check_weights(grouped.grouped_linear_weight_gradient(x, dy, bad), x, dy, keys)


@pytest.mark.parametrize("dtype,rows,k,n", [(F32, 9000, 96, 160), (F32, 9000, 300, 260), (BF16, 20_000, 264, 1096), (F16, 9000, 1025, 515)])
def test_captured_calls_and_another_stream(dtype, rows, k, n):
    """A captured run of grouping, product and gradients, replayed on new inputs while another stream runs its own."""
    from fastmace_b200 import grouped
    grouped.prepare_device()
    g = torch.Generator(device="cuda").manual_seed(9)

    def inputs():
        return (torch.randint(0, 6, (rows,), generator=g, device="cuda", dtype=torch.int32),
                torch.randn(rows, k, generator=g, device="cuda").to(dtype), torch.randn(6, k, n, generator=g, device="cuda").to(dtype),
                torch.randn(rows, n, generator=g, device="cuda").to(dtype))

    def calls(keys, x, w, dy):
        plan = grouped.group_rows(keys, 6)
        return (grouped.grouped_linear(x, w, plan), grouped.grouped_linear_input_gradient(dy, w, plan),
                grouped.grouped_linear_weight_gradient(x, dy, plan))

    held = inputs()
    calls(*held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = calls(*held)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        captured_too = calls(*held)
    side = torch.cuda.Stream()
    for _ in range(3):
        fresh, other = inputs(), inputs()
        for t, new in zip(held, fresh):
            t.copy_(new)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            beside = calls(*other)
            second.replay()
        graph.replay()
        torch.cuda.synchronize()
        for a, b, c in zip(captured, captured_too, calls(*fresh)):
            assert torch.equal(a, c) and torch.equal(b, c)
        for a, c in zip(beside, calls(*other)):
            assert torch.equal(a, c)
    grouped.check_status()


@pytest.mark.parametrize("dtype,k,n", [(F32, 128, 128), (F32, 200, 140), (BF16, 1032, 1040), (BF16, 264, 1096), (BF16, 130, 515)])
def test_weight_gradients_add_up(dtype, k, n):
    """accumulate=True over groups of one unit, of several and of none."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(12)
    keys = torch.cat([torch.zeros(3, dtype=torch.int32), torch.full((2990,), 2, dtype=torch.int32), torch.full((7,), 4, dtype=torch.int32)]).cuda()
    keys = keys[torch.randperm(3000, generator=g, device="cuda")]
    plan = grouped.group_rows(keys, 5)
    x = torch.randn(3000, k, generator=g, device="cuda").to(dtype)
    dy = torch.randn(3000, n, generator=g, device="cuda").to(dtype)
    base = torch.randn(5, k, n, generator=g, device="cuda")
    out = base.clone()
    assert grouped.grouped_linear_weight_gradient(x, dy, plan, out=out, accumulate=True) is out
    _check_weights(out, x, dy, keys, base=base)
    assert torch.equal(out[[1, 3]], base[[1, 3]])


def test_offsets_beyond_32_bits():
    """A row further than 2^31 elements into its array."""
    from fastmace_b200 import grouped
    rows, far = 40, 1 << 27
    need = rows * far * 2
    if torch.cuda.mem_get_info()[0] < 2 * need:
        pytest.skip("not enough memory")
    for k in (64, 33):
        x = torch.empty(rows * far, dtype=BF16, device="cuda").as_strided((rows, k), (far, 1))
        g = torch.Generator(device="cuda").manual_seed(10)
        x.copy_(torch.randn(rows, k, generator=g, device="cuda"))
        w = torch.randn(2, k, 64, generator=g, device="cuda").to(BF16)
        dy = torch.randn(rows, 64, generator=g, device="cuda").to(BF16)
        keys = torch.arange(rows, device="cuda") % 2
        plan = grouped.group_rows(keys, 2)
        _check_rows(grouped.grouped_linear(x, w, plan), x, w, keys)
        _check_weights(grouped.grouped_linear_weight_gradient(x, dy, plan), x, dy, keys)
        grouped.grouped_linear_input_gradient(dy, w, plan, out=x)
        _check_rows(x, dy, w, keys, transposed=True)


def test_refusals_on_the_device():
    from fastmace_b200 import grouped
    x, w = torch.zeros(8, 16, device="cuda"), torch.zeros(2, 16, 8, device="cuda")
    plan = grouped.group_rows(torch.zeros(8, dtype=torch.int32, device="cuda"), 2)
    for bad in (lambda: grouped.grouped_linear(x, w.half(), plan), lambda: grouped.grouped_linear(x[:, :15], w, plan),
                lambda: grouped.grouped_linear(x[:7], w, plan), lambda: grouped.grouped_linear(x, w[:1], plan),
                lambda: grouped.grouped_linear(x.double(), w.double(), plan), lambda: grouped.grouped_linear(x.t(), w, plan),
                lambda: grouped.grouped_linear(x, w.transpose(1, 2), plan), lambda: grouped.grouped_linear(x[:, :0], w[:, :0], plan),
                lambda: grouped.grouped_linear(x, w, plan, out=torch.zeros(8, 9, device="cuda")),
                lambda: grouped.grouped_linear(x, w, plan, out=torch.zeros(1, 8, device="cuda").expand(8, 8)),
                lambda: grouped.grouped_linear_weight_gradient(x, x[:7], plan),
                lambda: grouped.grouped_linear_weight_gradient(x, x, plan, accumulate=True),
                lambda: grouped.grouped_linear_weight_gradient(x, x, plan, out=torch.zeros(2, 16, 15, device="cuda")),
                lambda: grouped.grouped_linear_weight_gradient(x, x, plan, out=torch.zeros(1, 16, 16, device="cuda").expand(2, 16, 16)),
                lambda: grouped.grouped_linear_weight_gradient(x, x, plan, out=torch.zeros(40, device="cuda").as_strided((2, 16, 16), (1, 1, 1))),
                lambda: grouped.group_rows(torch.zeros(8, device="cuda"), 2),
                lambda: grouped.group_rows(torch.zeros(8, dtype=torch.int32, device="cuda"), 1025)):
        with pytest.raises(ValueError):
            bad()


def test_outputs_that_share_memory_with_operands():
    from fastmace_b200 import grouped
    nodes = torch.randn(40, 4, 64, device="cuda")
    w = torch.randn(2, 64, 64, device="cuda")
    keys = torch.arange(40, device="cuda") % 2
    plan = grouped.group_rows(keys, 2)
    for call in (lambda: grouped.grouped_linear(nodes[:, 0], w, plan, out=nodes[:, 0]),
                 lambda: grouped.grouped_linear_input_gradient(nodes[:, 0], w, plan, out=w.view(-1)[:2560].view(40, 64)),
                 lambda: grouped.grouped_linear_weight_gradient(nodes[:, 0], nodes[:, 1], plan, out=nodes.view(-1)[:8192].view(2, 64, 64))):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    # another component of the same array is no overlap
    before = nodes.clone()
    grouped.grouped_linear(nodes[:, 0], w, plan, out=nodes[:, 2])
    _check_rows(nodes[:, 2], before[:, 0], w, keys)
    assert torch.equal(nodes[:, 0], before[:, 0]) and torch.equal(nodes[:, 1], before[:, 1]) and torch.equal(nodes[:, 3], before[:, 3])


def test_graphs_that_saved_a_given_output_find_out():
    from fastmace_b200 import grouped
    x, dy, w = torch.ones(8, 16, device="cuda"), torch.ones(8, 8, device="cuda"), torch.ones(2, 16, 8, device="cuda")
    plan = grouped.group_rows(torch.zeros(8, dtype=torch.int32, device="cuda"), 2)
    for call, shape in ((lambda out: grouped.grouped_linear(x, w, plan, out=out), (8, 8)),
                        (lambda out: grouped.grouped_linear_input_gradient(dy, w, plan, out=out), (8, 16)),
                        (lambda out: grouped.grouped_linear_weight_gradient(x, dy, plan, out=out, accumulate=True), (2, 16, 8))):
        out = torch.zeros(shape, device="cuda")
        factor = torch.ones(shape, device="cuda", requires_grad=True)
        saved = (factor * out).sum()
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
    with torch.inference_mode():
        out = torch.zeros(8, 8, device="cuda")
        assert bool((grouped.grouped_linear(x, w, plan, out=out) == 16).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,groups,k,n", [(90, 3, 13, 21), (300, 2, 65, 129), (700, 5, 130, 515), (9, 4, 515, 301), (5000, 2, 263, 391),
                                             (3000, 40, 1026, 1030)])
def test_what_lies_beside_operands_and_outputs(rows, groups, k, n, dtype):
    """Rows at multiples of 16 bytes whose lengths are none: what is behind the end of a row of an operand (NaN here) takes no part,
    and behind that of an output stays as it was."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(k)
    keys = torch.randint(-1, groups, (rows,), generator=g, device="cuda", dtype=torch.int32)
    plan = grouped.group_rows(keys, groups)

    def room(*shape, fill, dtype=dtype):
        return torch.full((*shape[:-1], (shape[-1] + 15) // 8 * 8), fill, dtype=dtype, device="cuda")

    def within(*shape, scale=1.0):
        t = room(*shape, fill=float("nan"))[..., :shape[-1]]
        return t.copy_(torch.randn(*shape, generator=g, device="cuda") * scale)

    x, dy, w = within(rows, k), within(rows, n), within(groups, k, n, scale=k ** -0.5)
    y, dx, dw = room(rows, n, fill=7.0), room(rows, k, fill=7.0), room(groups, k, n, fill=7.0, dtype=F32)
    grouped.grouped_linear(x, w, plan, out=y[:, :n])
    grouped.grouped_linear_input_gradient(dy, w, plan, out=dx[:, :k])
    grouped.grouped_linear_weight_gradient(x, dy, plan, out=dw[:, :, :n])
    live = keys >= 0
    _check_rows(y[live][:, :n], x[live], w, keys[live])
    _check_rows(dx[live][:, :k], dy[live], w, keys[live], transposed=True)
    _check_weights(dw[:, :, :n], x, dy, keys)
    for t, width in ((y, n), (dx, k), (dw, n)):
        assert bool((t[..., width:] == 7).all())
    grouped.check_status()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [13, 64, 200, 515])
@pytest.mark.parametrize("wide", [(8, 21), (3, 2), (4, 0), (1, 8)])
def test_weights_of_one_row_cut_from_wider_ones(dtype, n, wide):
    """k == 1: the distance between the rows of a matrix, which nothing uses, may be anything; that between matrices as well."""
    from fastmace_b200 import grouped
    deep, more = wide
    g = torch.Generator(device="cuda").manual_seed(n + deep)
    keys = torch.randint(-1, 3, (70,), generator=g, device="cuda", dtype=torch.int32)
    plan = grouped.group_rows(keys, 3)
    w = torch.randn(3, deep, n + more, generator=g, device="cuda").to(dtype)[:, :1, :n]
    x = torch.randn(70, 1, generator=g, device="cuda").to(dtype)
    dy = torch.randn(70, n, generator=g, device="cuda").to(dtype)
    _check_rows(grouped.grouped_linear(x, w, plan), x, w, keys)
    _check_rows(grouped.grouped_linear_input_gradient(dy, w, plan), dy, w, keys, transposed=True)
    room = torch.full((3, deep, n + more), 7.0, device="cuda")
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan, out=room[:, :1, :n])
    _check_weights(dw, x, dy, keys)
    assert bool((room[:, 1:] == 7).all()) and bool((room[:, :, n:] == 7).all())
    grouped.check_status()


@pytest.mark.parametrize("rows,k,n", [(200, 64, 96), (200, 128, 200), (200, 300, 96), (8, 4096, 136), (70, 13, 21)])
def test_infinities_in_fp32_give_what_the_plain_product_gives(rows, k, n):
    """Infinities of both signs, NaN and zeros opposite to them, in rows and in weights; half of the finite values have eight significant
    bits at most, so that the lower parts of their splits are zeros. Where float64 has a number the others keep the usual bound."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(k)
    keys = torch.arange(rows, device="cuda") % 2
    plan = grouped.group_rows(keys, 2)
    inf, nan = float("inf"), float("nan")

    def values(*shape):
        t = torch.randn(*shape, generator=g, device="cuda")
        t[..., ::2] = t[..., ::2].to(BF16).float()
        return t

    def check(got, a, b):
        ref = a.double() @ b.double()
        fine = torch.isfinite(ref)
        assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got.isinf(), ref.isinf())
        assert torch.equal(got[got.isinf()].double(), ref[got.isinf()])
        assert bool(((got.double() - ref).abs() <= (a.shape[1] + 8) * 2.0 ** -24 * (a.double().abs() @ b.double().abs()))[fine].all())

    x, dy, w = values(rows, k), values(rows, n), values(2, k, n)
    for t in (x, dy):
        t[0, 2], t[1, 6], t[2, 7], t[3, 3], t[4, 5] = inf, -inf, nan, inf, -inf
        t[5, 2], t[5, 4] = inf, inf
        t[6, 2], t[6, 4] = inf, -inf
    w[0, 2, :9:2], w[1, 6, 1:8:3], w[:, 3, 11], w[:, 10, 5] = 0.0, 0.0, inf, -inf
    for each, kept in ((w, w.clone()), (torch.ones_like(w), torch.ones_like(w))):
        y, dx = grouped.grouped_linear(x, each, plan), grouped.grouped_linear_input_gradient(dy, each, plan)
        for q in range(2):
            check(y[keys == q], x[keys == q], kept[q])
            check(dx[keys == q], dy[keys == q], kept[q].t())
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan)
    for q in range(2):
        check(dw[q], x[keys == q].t(), dy[keys == q])
    grouped.check_status()


@pytest.mark.parametrize("size", [-105, -112, -120, -126, -132])
@pytest.mark.parametrize("k", [64, 300, 2100])
def test_smallest_fp32_operands_against_large_ones(size, k):
    """Products that are ordinary numbers of operands about 2^size and 2^60. The last of the three bf16 parts of a value ends at 2^-133,
    bf16's smallest number: up to that much of each value is lost, times what it is multiplied by, beside the usual bound."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(k)
    keys = torch.arange(40, device="cuda") % 2
    plan = grouped.group_rows(keys, 2)
    small = torch.randn(40, k, generator=g, device="cuda") * 2.0 ** -60 * 2.0 ** (size + 60)
    w = torch.randn(2, k, 200, generator=g, device="cuda") * 2.0 ** 60
    large = torch.randn(40, 200, generator=g, device="cuda") * 2.0 ** 60
    y, dw = grouped.grouped_linear(small, w, plan), grouped.grouped_linear_weight_gradient(small, large, plan)
    for q in range(2):
        for got, a, b in ((y[keys == q], small[keys == q], w[q]), (dw[q], small[keys == q].t(), large[keys == q])):
            a, b = a.double(), b.double()
            tol = (a.shape[1] + 8) * 2.0 ** -24 * (a.abs() @ b.abs()) + 2.0 ** -133 * b.abs().sum(0)
            assert bool(((got.double() - a @ b).abs() <= tol).all())


@pytest.mark.parametrize("dtype,k", [(F32, 2048), (F32, 256), (F32, 64), (BF16, 2048), (BF16, 64)])
def test_every_launch_is_counted(dtype, k):
    """Single tokens, with and without clusters that share the depth: one kernel a linear."""
    from fastmace_b200 import _lib, grouped
    lib = _lib.load()
    plan = grouped.group_rows(torch.arange(8, device="cuda"), 8)
    x, w = torch.ones(8, k, dtype=dtype, device="cuda"), torch.ones(8, k, 1024, dtype=dtype, device="cuda")
    before = lib.fmb_launch_count()
    grouped.grouped_linear(x, w, plan)
    assert lib.fmb_launch_count() == before + 1


@pytest.mark.parametrize("rows,groups,k,n", [(1500, 3, 128, 128), (1500, 3, 200, 136), (900, 2, 1032, 264), (600, 2, 2056, 136), (700, 2, 96, 4096),
                                             (8, 8, 2048, 1024), (1, 1, 4096, 40), (30, 1, 4096, 256), (40, 2, 515, 301)])
def test_fp32_operands_keep_their_bits_at_any_depth(rows, groups, k, n):
    """A bound on the norm, which does not grow with the depth as the bound per element does. An accumulator takes 16 additions before it moves
    to fp32, each cut off: up to 2^-23 of a partial sum, half of that on average, and partial sums are two thirds of the whole in the
    root mean square: 16 x 2^-24 x 0.7 = 6.7e-7. The products left out are 2^-23 of the terms at most, the sums of chunks are rounded a
    few times: 1e-6 in all. Operands of 16 significant bits would be off by 2^-17 of each term, 5e-6 of the norm, tf32 by 2e-4. The splits
    of few rows among several blocks of a cluster, from a depth of 512 on, are the same sums."""
    from fastmace_b200 import grouped
    g = torch.Generator(device="cuda").manual_seed(k)
    keys = torch.arange(rows, device="cuda") % groups
    plan = grouped.group_rows(keys, groups)
    x, dy = (torch.randn(rows, width, generator=g, device="cuda") for width in (k, n))
    w = torch.randn(groups, k, n, generator=g, device="cuda")
    y, dx = grouped.grouped_linear(x, w, plan), grouped.grouped_linear_input_gradient(dy, w, plan)
    dw = grouped.grouped_linear_weight_gradient(x, dy, plan)
    for q in range(groups):
        r = keys == q
        a, b, c = x[r].double(), dy[r].double(), w[q].double()
        for got, ref in ((y[r], a @ c), (dx[r], b @ c.t()), (dw[q], a.t() @ b)):
            assert float((got.double() - ref).norm()) <= 1e-6 * float(ref.norm())
