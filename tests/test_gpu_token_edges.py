"""Calls of embedding rows, held rows and experts at the edges of what they take: rows and matrices further apart than 32 bits reach, the
longest rows, slices of what is held, all choices alike, work on other streams ahead of a launch, first calls inside a capture."""
import os
import subprocess
import sys

import pytest
import torch
from conftest import ROOT

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
FAR = 2 ** 30 + 40                              # values between rows: the third starts past 2^31 of them, and past 2^32 bytes


def _far(rows):
    """The same rows, FAR apart."""
    big = torch.empty((len(rows) - 1) * FAR + rows.shape[1] + 8, dtype=rows.dtype, device="cuda")
    view = big.as_strided(rows.shape, (FAR, 1))
    view.copy_(rows)
    return view


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_past_32_bits(dtype):
    from fastmace_b200 import checkpoints, embedding, experts
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(3, 72, generator=g, device="cuda").to(dtype)
    far = _far(rows)
    tokens = torch.tensor([2, 0, 5, 1, 2], device="cuda")
    assert torch.equal(embedding.embedding(tokens, far, 2.0), embedding.embedding(tokens, rows, 2.0))
    out = _far(torch.zeros_like(rows))
    embedding.embedding(tokens[:3], rows, 2.0, out=out)
    assert torch.equal(out[:2], embedding.embedding(tokens[:2], rows, 2.0)) and bool((out[2] == 0).all())
    order = embedding.sort_tokens(torch.tensor([1, 1, 0], device="cuda"), 3)
    assert torch.equal(embedding.embedding_gradient(far, order, 3), embedding.embedding_gradient(rows, order, 3))
    held, want = checkpoints.hold_rows(far, parts=2), checkpoints.hold_rows(rows, parts=2)
    assert torch.equal(held.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(held.exponents, want.exponents)
    checkpoints.release_rows(held, out=out)
    assert torch.equal(out, checkpoints.release_rows(want))
    assert torch.equal(checkpoints.gated_rows(far), checkpoints.gated_rows(rows))
    dh = torch.randn(3, 36, generator=g, device="cuda").to(dtype)
    checkpoints.gated_rows_gradient(held, dh, out=out)
    assert torch.equal(out, checkpoints.gated_rows_gradient(want, dh)[0])
    router = torch.randn(72, 5, generator=g, device="cuda").to(dtype)
    routes, again = experts.route_rows(far, router, 2), experts.route_rows(rows, router, 2)
    assert torch.equal(routes.experts, again.experts) and torch.equal(routes.weights, again.weights)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradient_rows_and_experts_past_32_bits(dtype):
    from fastmace_b200 import embedding, experts
    g = torch.Generator(device="cuda").manual_seed(2)
    order = embedding.sort_tokens(torch.randint(0, 3, (5000,), generator=g, device="cuda"), 3)
    dy = torch.randn(5000, 72, generator=g, device="cuda").to(dtype)
    want = embedding.embedding_gradient(dy, order, 3)
    out = _far(torch.ones(3, 72, device="cuda"))
    embedding.embedding_gradient(dy, order, 3, out=out)
    assert torch.equal(out, want)
    del out
    x = torch.randn(4, 72, generator=g, device="cuda").to(dtype)
    up, down = (torch.randn(3, *s, generator=g, device="cuda").to(dtype) / 8 for s in ((72, 80), (40, 72)))
    routes = experts.route_rows(x, torch.randn(72, 3, generator=g, device="cuda").to(dtype), 3)
    want = experts.expert_layer(x, up, down, routes)
    far = [_far(w.reshape(3, -1)).as_strided(w.shape, (FAR, w.shape[2], 1)) for w in (up, down)]
    assert torch.equal(experts.expert_layer(x, *far, routes), want)
    del far
    assert torch.equal(experts.expert_layer(x, up, down, routes, out=_far(want)), want)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width,inner", [(131_072, 5), (8, 131_072), (131_071, 3), (9, 131_071)])
def test_the_longest_rows_of_a_layer(width, inner, dtype):
    from fastmace_b200 import experts
    from test_gpu_experts import _check, _layer
    g = torch.Generator(device="cuda").manual_seed(inner)
    x, up, down = _layer(9, 2, width, inner, dtype, g)
    chosen, weights = torch.tensor([[0], [1], [1]] * 3, dtype=torch.int32, device="cuda"), torch.rand(9, 1, generator=g, device="cuda")
    _check(experts.expert_layer(x, up, down, experts.Routes(chosen, weights)), x, up, down, chosen, weights)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_all_pairs_at_one_expert_and_one_matrix_for_all(dtype):
    from fastmace_b200 import experts
    from test_gpu_experts import _check, _layer
    g = torch.Generator(device="cuda").manual_seed(7)
    x, up, down = _layer(128, 5, 70, 33, dtype, g)
    weights = torch.randn(128, 16, generator=g, device="cuda") / 4
    chosen = torch.full((128, 16), 3, dtype=torch.int32, device="cuda")
    _check(experts.expert_layer(x, up, down, experts.Routes(chosen, weights)), x, up, down, chosen, weights)
    # expanded weights: every expert's are the same
    chosen = torch.randint(0, 5, (128, 16), generator=g, device="cuda", dtype=torch.int32)
    shared = [w[:1].expand(5, -1, -1) for w in (up, down)]
    y = experts.expert_layer(x, *shared, experts.Routes(chosen, weights))
    assert torch.equal(y, experts.expert_layer(x, *(w.contiguous() for w in shared), experts.Routes(chosen, weights)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("columns", [64, 66, 515, 35])
def test_slices_of_held_rows(columns, dtype):
    """Codes that begin at any byte."""
    from fastmace_b200 import checkpoints, grouped
    g = torch.Generator(device="cuda").manual_seed(columns)
    x = torch.randn(203, columns, generator=g, device="cuda").to(dtype)
    for parts in (1, 2) if columns % 2 == 0 else (1,):
        held = checkpoints.hold_rows(x, parts)
        back = checkpoints.release_rows(held)
        for first in (1, 2, 3, 5):
            part = checkpoints.HeldRows(held.codes[first:], held.exponents[first:], held.dtype, parts)
            assert torch.equal(checkpoints.release_rows(part), back[first:])
            if parts == 2:
                dh = torch.randn(203 - first, columns // 2, generator=g, device="cuda").to(dtype)
                got, want = checkpoints.gated_rows_gradient(part, dh), checkpoints.gated_rows_gradient(back[first:].contiguous(), dh)
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            else:
                dy = torch.randn(203 - first, 24, generator=g, device="cuda").to(dtype)
                plan = grouped.group_rows(torch.randint(0, 3, (203 - first,), generator=g, device="cuda"), 3)
                copy = checkpoints.HeldRows(part.codes.clone(), part.exponents.clone(), held.dtype, 1)
                assert torch.equal(checkpoints.held_weight_gradient(part, dy, plan), checkpoints.held_weight_gradient(copy, dy, plan))


def test_work_of_another_stream_ahead_of_an_early_launch():
    """A launch that comes early waits for an event between it and the launch before, which has said that others may come."""
    from fastmace_b200 import embedding, experts
    g = torch.Generator(device="cuda").manual_seed(3)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    heavy = torch.randn(2048, 2048, generator=g, device="cuda")
    few, many = torch.randint(0, 500, (4000,), generator=g, device="cuda"), torch.randint(0, 500, (20_000,), generator=g, device="cuda")
    x = torch.randn(16, 256, generator=g, device="cuda").to(BF16)
    up, down = (torch.randn(8, *s, generator=g, device="cuda").to(BF16) / 16 for s in ((256, 128), (64, 256)))
    weights = torch.rand(16, 2, generator=g, device="cuda")
    dy = torch.randn(20_000, 40, generator=g, device="cuda")
    chosen, tokens = torch.zeros(16, 2, dtype=torch.int32, device="cuda"), torch.zeros(20_000, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    for n in range(12):
        new, fresh = torch.randint(0, 8, (16, 2), generator=g, device="cuda", dtype=torch.int32), torch.randint(0, 500, (20_000,), generator=g, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(b):
            for _ in range(3):
                heavy = heavy @ heavy / 2048
            chosen.copy_(new)
            tokens.copy_(fresh)
            done = b.record_event()
        with torch.cuda.stream(a):
            embedding.sort_tokens(few, 500)       # its kernel lets the next one come
            a.wait_event(done)
            if n % 2:
                y = experts.expert_layer(x, up, down, experts.Routes(chosen, weights))
                order = embedding.sort_tokens(tokens, 500)
            else:
                order = embedding.sort_tokens(tokens, 500)
                y = experts.expert_layer(x, up, down, experts.Routes(chosen, weights))
            grad = embedding.embedding_gradient(dy, order, 500)
        torch.cuda.synchronize()
        assert torch.equal(y, experts.expert_layer(x, up, down, experts.Routes(new, weights)))
        want = embedding.sort_tokens(fresh, 500)
        assert torch.equal(order.rows, want.rows) and torch.equal(grad, embedding.embedding_gradient(dy, want, 500))
        b.wait_stream(a)


FIRST = """
import sys, torch
from fastmace_b200 import checkpoints, embedding, experts
x = torch.arange(8 * 64, device="cuda").view(8, 64).to(torch.bfloat16) / 512
tokens = torch.arange(8, device="cuda")
big = torch.arange(20000, device="cuda") % 3000
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    y = embedding.embedding(tokens, x, 2.0)
    order = embedding.sort_tokens(big, 3000)
    few = embedding.embedding_gradient(x, embedding.sort_tokens(tokens, 8), 8)
    h, held = checkpoints.gated_rows(x, hold=True)
    back = checkpoints.release_rows(checkpoints.hold_rows(x))
    du, again = checkpoints.gated_rows_gradient(held, h)
    routes = experts.route_rows(x, x.t().contiguous(), 3)
    more = experts.route_rows(x.repeat(30, 1), x.t().contiguous(), 3)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, 2 * x) and torch.equal(few, x.float()) and torch.equal(order.keys, big.sort().values.int())
want = experts.route_rows(x, x.t().contiguous(), 3)
assert torch.equal(routes.experts, want.experts) and torch.equal(more.experts[:8], experts.route_rows(x.repeat(30, 1), x.t().contiguous(), 3).experts[:8])
assert torch.equal(du, checkpoints.gated_rows_gradient(held, h)[0]) and torch.equal(back, checkpoints.release_rows(checkpoints.hold_rows(x)))
print("captured first")
"""


def test_first_calls_of_a_process_may_be_captured():
    run = subprocess.run([sys.executable, "-c", FIRST], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured first" in run.stdout, run.stderr[-2000:]
