"""AdamW on the GPU against the formula in float64.

Tolerances of one step. With moments in 32 bits m and v are one product and one fused or rounded sum of two terms: 4 roundings,
2^-22 of the terms' magnitudes. A weight moves by at most a few lr, computed with about ten roundings and an approximate
division (2^-22): 2^-20 of the update, and one rounding of the weight, 2^-24 of it (plus 2^-24 for the decay's). Moments in 8 bits: the
new moment is within half a step of e4m3 of the formula's, 2^-4 of itself or 2^-10 of the block's scale (below its smallest normal
number), and the scale is off by a rounding or two, 2^-22.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

SIZES = [[1], [5, 300, 256, 255, 257, 1000], [16_384, 4096, 512, 2, 33_000], [3] * 450, [200_001]]


def _formula(p, g, m, v, t, lr, b1, b2, eps, wd):
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = lr / (1 - b1 ** t) * m / (torch.sqrt(v) / (1 - b2 ** t) ** 0.5 + eps)
    return p * (1 - lr * wd) - update, m, v, update


def _case(sizes, grad, seed, offset=0):
    """Weights and gradients of the sizes, views of one buffer each that start `offset` elements off its alignment."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = sum(sizes)

    def views(t):
        out, at = [], offset
        for n in sizes:
            out.append(t[at:at + n])
            at += n
        return out

    p = torch.randn(total + offset, generator=g, device="cuda")
    size = torch.exp(3 * torch.randn(total + offset, generator=g, device="cuda")) * 1e-3
    gr = (torch.randn(total + offset, generator=g, device="cuda") * size).to(grad)
    return views(p), views(gr), views(torch.zeros(total + offset, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_steps_against_the_formula(sizes, bits, grad, offset):
    from fastmace_b200.optimiser import BLOCK, AdamW
    hyper = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)
    params, _, copies = _case(sizes, grad, 1, offset)
    opt = AdamW(params, state_bits=bits, copies=copies, **hyper)
    for t in range(1, 4):
        grads = _case(sizes, grad, 10 + t, offset)[1]
        before = [(p.double(), *(x.double() for x in opt.moments(k))) for k, p in enumerate(params)]
        opt.step(grads)
        for k, (p, g, c) in enumerate(zip(params, grads, copies)):
            p0, m0, v0 = before[k]
            rp, rm, rv, update = _formula(p0, g.double(), m0, v0, t, 3e-3, 0.9, 0.99, 1e-8, 0.02)
            assert bool(((p.double() - rp).abs() <= 2.0 ** -20 * update.abs() + 2.0 ** -23 * p0.abs() + 1e-30).all())
            assert torch.equal(c, p.to(torch.bfloat16))
            m, v = (x.double() for x in opt.moments(k))
            if bits == 32:
                assert bool(((m - rm).abs() <= 2.0 ** -22 * (0.9 * m0.abs() + 0.1 * g.double().abs()) + 1e-37).all())
                assert bool(((v - rv).abs() <= 2.0 ** -22 * rv + 1e-37).all())
                continue
            blocks = -(-p.numel() // BLOCK)
            for got, ref in ((m, rm), (v.sqrt(), rv.sqrt())):
                pad = torch.zeros(blocks * BLOCK, dtype=torch.float64, device="cuda")
                pad[:p.numel()] = ref.view(-1)
                scale = (pad.view(-1, BLOCK).abs().amax(1) / 448).repeat_interleave(BLOCK)[:p.numel()]
                tol = torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * scale) * (1 + 2.0 ** -18) + 2.0 ** -135
                # a root too small for the type is held as the smallest number, 2^-9 of the scale, instead of zero
                if got is not m:
                    tol = torch.where((ref > 0) & (ref < 2.0 ** -9 * scale), 2.0 ** -9 * scale, tol)
                assert bool(((got - ref).abs() <= tol).all()), float(((got - ref).abs() - tol).max())
            assert bool((v[rv > 0] > 0).all())
    assert opt.steps == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_a_gradient_stay(bits):
    from fastmace_b200.optimiser import AdamW
    g = torch.Generator(device="cuda").manual_seed(3)
    weights = {n: torch.randn(s, generator=g, device="cuda") for n, s in (("a", (7, 90)), ("b", (300,)), ("c", (4, 5, 6)), ("d", (0,)))}
    opt = AdamW(weights, lr=0.1, state_bits=bits)
    opt.step({n: torch.ones_like(w) for n, w in weights.items()})
    kept = [weights["b"].clone(), *opt.moments("b")]
    old = weights["a"].clone()
    opt.step({"a": torch.ones(7, 90, device="cuda"), "c": torch.ones(4, 5, 6, device="cuda"), "b": None})
    assert all(torch.equal(x, y) for x, y in zip(kept, (weights["b"], *opt.moments("b"))))
    assert not torch.equal(old, weights["a"]) and opt.steps == 2
    opt.step({})
    assert opt.steps == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """A captured step replayed with new gradients gives the bits of the same steps taken one by one, and two optimisers' graphs
    replayed on two streams do not meet."""
    from fastmace_b200.optimiser import AdamW
    g = torch.Generator(device="cuda").manual_seed(4)
    start = [torch.randn(n, generator=g, device="cuda") for n in (5000, 77, 300)]
    grads = [[torch.randn(n, generator=g, device="cuda") for n in (5000, 77, 300)] for _ in range(6)]

    def fresh():
        params = [p.clone() for p in start]
        return params, AdamW(params, lr=1e-2, state_bits=bits)

    params, opt = fresh()
    for step in grads:
        opt.step(step)
    runs = []
    for _ in range(2):
        p, o = fresh()
        held = [x.clone() for x in grads[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o.step(held)
        runs.append((p, o, held, graph, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for step in grads:
        for p, o, held, graph, stream in runs:
            with torch.cuda.stream(stream):
                for h, x in zip(held, step):
                    h.copy_(x)
                graph.replay()
    torch.cuda.synchronize()
    for p, o, *_ in runs:
        assert o.steps == 6 and all(torch.equal(a, b) for a, b in zip(p, params))
        assert torch.equal(o.m.view(torch.uint8), opt.m.view(torch.uint8)) and torch.equal(o.v.view(torch.uint8), opt.v.view(torch.uint8))


def test_continued_from_given_moments():
    from fastmace_b200.optimiser import AdamW
    for bits in (32, 8):
        g = torch.Generator(device="cuda").manual_seed(5)
        a = [torch.randn(1000, generator=g, device="cuda")]
        b = [a[0].clone()]
        grads = [[torch.randn(1000, generator=g, device="cuda")] for _ in range(4)]
        one, two = AdamW(a, state_bits=bits), AdamW(b, state_bits=bits)
        for x in grads:
            one.step(x)
        for x in grads[:2]:
            two.step(x)
        held = (two.m.clone(), two.v.clone()) if bits == 32 else (two.m.clone(), two.m_scale.clone(), two.v.clone(), two.v_scale.clone())
        two = AdamW(b, state_bits=bits)
        two.load_moments(2, *held)
        for x in grads[2:]:
            two.step(x)
        assert torch.equal(a[0], b[0]) and two.steps == 4


def test_values_that_are_not_finite_or_zero():
    from fastmace_b200.optimiser import AdamW
    for bits in (32, 8):
        p = [torch.ones(1024, device="cuda")]
        opt = AdamW(p, lr=0.1, weight_decay=0.0, state_bits=bits)
        opt.step([torch.zeros(1024, device="cuda")])
        assert bool((p[0] == 1).all())
        bad = torch.ones(1024, device="cuda")
        bad[300] = float("nan")
        bad[800] = float("inf")
        opt.step([bad])
        fine = torch.ones(1024, dtype=torch.bool, device="cuda")
        fine[[300, 800]] = False
        assert bool(torch.isfinite(p[0][fine]).all()) and bool(torch.isnan(p[0][300]))
        opt.step([torch.ones(1024, device="cuda")])
        if bits == 8:
            fine[256:512] = False
            fine[768:] = False
        assert bool(torch.isfinite(p[0][fine]).all()) and bool(torch.isnan(p[0][300])) and not bool(torch.isfinite(p[0][800]))


def test_refusals_on_the_device():
    from fastmace_b200.optimiser import AdamW
    w = torch.zeros(8, 8, device="cuda")
    for bad in (lambda: AdamW([]), lambda: AdamW([w.half()]), lambda: AdamW([w.t()[:4]]), lambda: AdamW([w], state_bits=16), lambda: AdamW([w, w]),
                lambda: AdamW([w], betas=(1.0, 0.9)), lambda: AdamW([w], lr=-1.0), lambda: AdamW([w], copies=[w]),
                lambda: AdamW([w], copies=[w.half()[:4]]), lambda: AdamW([w]).step([w, w]), lambda: AdamW([w]).step([w.double()]),
                lambda: AdamW([w]).step([w[:4]]), lambda: AdamW([w]).step([w.t()]), lambda: AdamW({"a": w}).step({"b": w}),
                lambda: AdamW([w, w.clone()]).step([w, w.half()]), lambda: AdamW([w]).step([w.cpu()]),
                lambda: AdamW([w]).load_moments(1, w), lambda: AdamW([w]).load_moments(1, w, w)):
        with pytest.raises(ValueError):
            bad()


def test_lists_that_share_memory_or_move():
    from fastmace_b200.optimiser import AdamW
    base = torch.zeros(1000, device="cuda")
    for bad in (lambda: AdamW([base[:600], base[500:]]), lambda: AdamW([base[:10], base[:10]]),
                lambda: AdamW([base[:500]], copies=[base[250:500].view(torch.bfloat16)]),
                lambda: AdamW([base[:10]], copies=[None, None]), lambda: AdamW({"a": base[:10]}, copies={"b": None})):
        with pytest.raises(ValueError):
            bad()
    optimiser = AdamW({"a": base[:500], "b": base[500:]}, copies={"b": torch.zeros(500, dtype=torch.float16, device="cuda")})
    optimiser.step({"a": torch.ones(500, device="cuda"), "b": torch.ones(500, device="cuda")})
    weight = torch.nn.Parameter(torch.ones(100, device="cuda"))
    optimiser = AdamW([weight])
    version = weight._version
    optimiser.step([torch.ones(100, device="cuda")])
    assert weight._version > version                      # a graph that saved the weights finds out
    weight.data = torch.ones(100, device="cuda")
    with pytest.raises(ValueError, match="other memory"):
        optimiser.step([torch.ones(100, device="cuda")])


@pytest.mark.parametrize("saved", ["plain", "copy", "asked later"])
def test_graphs_that_saved_a_weight_find_out(saved):
    """The gradient in the activations needs the weight that the product was made with, whether or not that asks for one itself."""
    from fastmace_b200.optimiser import AdamW
    weights = {n: torch.randn(16, 16, device="cuda") for n in "ab"}
    copies = {n: w.to(torch.bfloat16) for n, w in weights.items()}
    optimiser = AdamW(weights, copies=copies)
    if saved == "asked later":
        weights["a"].requires_grad_()
    used = {n: (copies if saved == "copy" else weights)[n] for n in "ab"}
    x = torch.randn(4, 16, device="cuda", dtype=used["a"].dtype, requires_grad=True)
    outputs = {n: (x @ w).sum() for n, w in used.items()}
    optimiser.step({"a": torch.ones(16, 16, device="cuda")})
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        outputs["a"].backward()
    outputs["b"].backward()                                # no gradient, no step
    # sums of 16 products with ones: 16 additions in fp32 in an order that is the library's, and the result's own rounding
    ref, size = used["b"].double().sum(1), used["b"].double().abs().sum(1)
    assert bool(((x.grad.double() - ref).abs() <= 16 * 2.0 ** -24 * size * 1.01 + torch.finfo(x.dtype).eps / 2 * size).all())


def test_tensors_of_inference_mode_are_stepped():
    from fastmace_b200.optimiser import AdamW
    with torch.inference_mode():
        weight = torch.ones(300, device="cuda")
        AdamW([weight]).step([torch.ones(300, device="cuda")])
        assert bool((weight < 1).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_of_a_captured_step_live_on(bits):
    """A captured step goes on with the moments it was captured with after others have been loaded: they stay allocated, and the loaded
    ones are not its."""
    import weakref

    from fastmace_b200.optimiser import AdamW
    weight, grad = torch.ones(1000, device="cuda"), torch.ones(1000, device="cuda")
    optimiser = AdamW([weight], state_bits=bits)
    optimiser.step([grad])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        optimiser.step([grad])
    names = ("m", "v") if bits == 32 else ("m", "m_scale", "v", "v_scale")
    old = [weakref.ref(getattr(optimiser, name)) for name in names]
    loaded = [getattr(optimiser, name).clone() for name in names]
    kept = [t.clone() for t in loaded]
    optimiser.load_moments(1, *loaded)
    assert all(ref() is not None for ref in old)
    before = [ref().clone() for ref in old]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(loaded, kept))
    assert any(not torch.equal(ref().view(torch.uint8), b.view(torch.uint8)) for ref, b in zip(old, before))
    # without a captured step nothing is kept
    other = AdamW([torch.ones(1000, device="cuda")], state_bits=bits)
    gone = weakref.ref(other.m)
    other.load_moments(1, *(t.clone() for t in loaded))
    assert gone() is None


def test_a_copy_that_moved_is_refused():
    """As a weight that moved: the step would write to where the copy was, which lives on all the same."""
    from fastmace_b200.optimiser import AdamW
    weights = [torch.ones(300, device="cuda"), torch.ones(5, device="cuda")]
    copy = torch.zeros(300, dtype=torch.bfloat16, device="cuda")
    optimiser = AdamW(weights, copies=[copy, None])
    optimiser.step([torch.ones_like(w) for w in weights])
    assert torch.equal(copy, weights[0].to(torch.bfloat16))
    place, storage = copy.data_ptr(), torch.empty(300, dtype=torch.bfloat16, device="cuda")
    copy.data = storage
    taken = [torch.empty(300, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
    assert all(t.data_ptr() != place for t in taken)
    with pytest.raises(ValueError, match="other memory"):
        optimiser.step([torch.ones_like(w) for w in weights])


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_that_share_memory_are_refused(bits):
    from fastmace_b200.optimiser import AdamW
    weight = torch.ones(512, device="cuda")
    optimiser = AdamW([weight], state_bits=bits)
    names = ("m", "v") if bits == 32 else ("m", "m_scale", "v", "v_scale")
    fine = {name: getattr(optimiser, name).clone() for name in names}
    room = torch.zeros(1000, dtype=fine["m"].dtype, device="cuda")
    bad = [{**fine, "v": fine["m"]}, {**fine, "m": room[:512], "v": room[256:768]}]
    bad.append({**fine, "m": weight} if bits == 32 else {**fine, "v_scale": weight[:2]})
    for moments in bad:
        with pytest.raises(ValueError, match="share"):
            optimiser.load_moments(1, *moments.values())
    for steps in (-1, 2.5):
        with pytest.raises(ValueError):
            optimiser.load_moments(steps, *fine.values())
    optimiser.load_moments(1, *fine.values())
    optimiser.step([torch.ones(512, device="cuda")])
    assert optimiser.steps == 2


@pytest.mark.parametrize("course", ["steady", "sizes drawn anew", "half fall to a tenth"])
def test_second_moments_in_8_bits_follow_those_in_32(course):
    """Thousands of steps of random gradients, whose sizes change on the way. At random rounding the expected v is that of 32 bits. A
    root changes by no more than 1/2,000 of itself a step downwards (and as much upwards on average); a change of c between codes d apart, d at most
    1/8 of the value, adds a variance of d c at most, which fades by 1/1,000 a step: 1/8 x 1/2,000 x 1,000 = 1/16, a spread of a quarter
    at most, and nine values in ten within 1.65 of that. The sum of v over 262,144 values whose sizes are lognormals of e^0.5 then spreads by
    0.2 %. First moments are rounded to the nearest: they are compared with nothing here."""
    from fastmace_b200.optimiser import AdamW
    n = 262_144
    g = torch.Generator(device="cuda").manual_seed(7)
    sizes = [torch.exp(0.5 * torch.randn(n, generator=g, device="cuda"))]
    if course == "steady":
        sizes.append(sizes[0])
    elif course == "sizes drawn anew":
        sizes.append(torch.exp(0.5 * torch.randn(n, generator=g, device="cuda")))
    else:
        sizes.append(sizes[0] * torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, 0.1, 1.0))
    weights = [torch.zeros(n, device="cuda") for _ in range(2)]
    optimisers = [AdamW([weights[0]], state_bits=8, rounding="random", seed=3), AdamW([weights[1]])]
    for step in range(5000):
        grad = torch.randn(n, generator=g, device="cuda") * sizes[step >= 1000]
        for optimiser in optimisers:
            optimiser.step([grad])
        if step in (100, 999, 4999):
            held, true = (optimiser.moments(0)[1].double() for optimiser in optimisers)
            low, high = torch.quantile((held / true).sqrt(), torch.tensor([0.05, 0.95], dtype=torch.float64, device="cuda")).tolist()
            assert 1 - 1.65 / 4 < low and high < 1 + 1.65 / 4, (step, low, high)
            assert abs(float(held.sum() / true.sum()) - 1) < 0.01, step


@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_one_step_rounded_at_random(sizes, grad):
    """Weights, first moments and scales are those of rounding to the nearest, bit by bit; a root is one of the two numbers of the type
    that its exact value lies between; v is exact on average over the seeds."""
    from fastmace_b200.optimiser import BLOCK, AdamW
    hyper = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02, state_bits=8)
    params, grads, copies = _case(sizes, grad, 1)
    start, first = [p.clone() for p in params], _case(sizes, grad, 5)[1]

    def run(**more):
        for p, s in zip(params, start):
            p.copy_(s)
        optimiser = AdamW(params, copies=copies, **hyper)
        optimiser.step(first)
        held = [t.clone() for t in (optimiser.m, optimiser.m_scale, optimiser.v, optimiser.v_scale)]
        optimiser = AdamW(params, copies=copies, **hyper, **more)
        optimiser.load_moments(1, *held)
        before = [optimiser.moments(k)[1].double() for k in range(len(params))]
        optimiser.step(grads)
        return optimiser, before, [p.clone() for p in params], [c.clone() for c in copies]

    nearest, before, weights, bf16 = run()
    total, seeds = 0.0, 24
    exact = torch.cat([0.99 * v + 0.01 * g.double().view(-1) ** 2 for v, g in zip(before, grads)])
    for seed in range(seeds):
        other, _, w, c = run(rounding="random", seed=seed)
        assert all(torch.equal(a, b) for a, b in zip(weights + bf16, w + c))
        assert torch.equal(nearest.m.view(torch.uint8), other.m.view(torch.uint8))
        assert torch.equal(nearest.m_scale, other.m_scale) and torch.equal(nearest.v_scale, other.v_scale)
        codes = torch.cat([other.v[b * BLOCK:b * BLOCK + p.numel()] for b, p in zip(other.blocks, params)]).double()
        scale = torch.cat([other.v_scale[b:b - (-p.numel() // BLOCK)].repeat_interleave(BLOCK)[:p.numel()]
                           for b, p in zip(other.blocks, params)]).double()
        unit = exact.sqrt() / scale
        gap = torch.exp2(torch.floor(torch.log2(torch.maximum(unit, codes).clamp(min=2.0 ** -6))) - 3)
        tiny = (unit < 2.0 ** -9) & (unit > 0)                      # held as the smallest number
        # (2^-21: the roots are fp32, and so are their quotients)
        assert bool(((codes - unit).abs() < gap + 2.0 ** -21 * unit)[~tiny].all()) and bool((codes[tiny] == 2.0 ** -9).all())
        total = total + torch.where(tiny, unit, codes) ** 2
    # independent errors of v in units of its scale: each spreads by half of what the squares of its two codes are apart, 2 unit gap, at most
    off, spread = (total / seeds - unit ** 2).sum(), float(((unit + gap) * gap).norm()) / seeds ** 0.5
    assert abs(float(off)) <= 6 * spread + 2.0 ** -20 * float((unit ** 2).sum())


def test_random_rounding_repeats_itself():
    """By seed, step and place: again, captured, continued, and whatever else is in the list behind."""
    from fastmace_b200.optimiser import AdamW
    g = torch.Generator(device="cuda").manual_seed(4)
    start = [torch.randn(n, generator=g, device="cuda") for n in (5000, 77, 300)]
    grads = [[torch.randn(n, generator=g, device="cuda") for n in (5000, 77, 300)] for _ in range(6)]

    def run(seed, mode="plain", count=3):
        params = [p.clone() for p in start[:count]]
        optimiser = AdamW(params, state_bits=8, rounding="random", seed=seed)
        if mode == "captured":
            held = [x.clone() for x in grads[0]]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                optimiser.step(held)
        for k, step in enumerate(grads):
            if mode == "captured":
                for h, x in zip(held, step):
                    h.copy_(x)
                graph.replay()
                continue
            if mode == "continued" and k == 3:
                held = [t.clone() for t in (optimiser.m, optimiser.m_scale, optimiser.v, optimiser.v_scale)]
                optimiser = AdamW(params, state_bits=8, rounding="random", seed=seed)
                optimiser.load_moments(3, *held)
            optimiser.step(step[:count])
        return params, optimiser.v.view(torch.uint8).clone()

    params, codes = run(5)
    for mode in ("plain", "captured", "continued"):
        p, c = run(5, mode)
        assert torch.equal(c, codes) and all(torch.equal(a, b) for a, b in zip(p, params)), mode
    p, c = run(5, count=1)
    assert torch.equal(c, codes[:len(c)]) and torch.equal(p[0], params[0])
    assert not torch.equal(run(6)[1], codes)


def test_random_rounding_of_values_that_are_not_finite_or_zero():
    from fastmace_b200.optimiser import AdamW
    weight = torch.ones(1024, device="cuda")
    optimiser = AdamW([weight], lr=0.1, weight_decay=0.0, state_bits=8, rounding="random")
    optimiser.step([torch.zeros(1024, device="cuda")])
    assert bool((weight == 1).all()) and bool((optimiser.v.float() == 0).all())
    bad = torch.ones(1024, device="cuda")
    bad[300], bad[800] = float("nan"), float("inf")
    for _ in range(2):
        optimiser.step([bad])
        bad = torch.ones(1024, device="cuda")
    fine = torch.ones(1024, dtype=torch.bool, device="cuda")
    fine[256:512], fine[768:] = False, False
    assert bool(torch.isfinite(weight[fine]).all()) and not bool(torch.isfinite(weight[[300, 800]]).any())
    assert bool(torch.isnan(optimiser.moments(0)[1][~fine]).all()) and bool(torch.isfinite(optimiser.moments(0)[1][fine]).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_lists_of_empty_tensors(bits):
    from fastmace_b200.optimiser import AdamW
    empty, weight = torch.zeros(0, 7, device="cuda"), torch.ones(3, device="cuda")
    optimiser = AdamW([empty, torch.zeros(0, device="cuda")], state_bits=bits)
    optimiser.step([torch.zeros(0, 7, device="cuda"), None])
    assert optimiser.steps == 0 and optimiser.moments(0)[0].shape == (0, 7)
    optimiser = AdamW([empty, weight], state_bits=bits)
    optimiser.step([torch.zeros(0, 7, device="cuda"), None])
    assert optimiser.steps == 0 and bool((weight == 1).all())
    optimiser.step([torch.zeros(0, 7, device="cuda"), torch.ones(3, device="cuda")])
    assert optimiser.steps == 1 and bool((weight < 1).all())
