"""The operators together, as a model of tokens is trained and served with them: embedding rows, routed experts by grouped products whose
inputs are kept in 8 bits, all gradients, an AdamW step; and the same layer for a few tokens in one call.

Tolerances, of norms. Every gradient is compared with the formulas in float64 on the values that are held, so what 8 bits lose is on both
sides. What is left are float32 sums (2^-20 of the terms' absolute sums with split operands, whose norms are at most 16 times the sums'
for the 24 to 256 terms of random sign here: 2^-16 a product, six in a row) and, in bfloat16, a rounding of 2^-8 at most of each result
in between, up to seven of them in a row.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
V, D, F, EXPERTS, TOP, T = 300, 64, 48, 6, 2, 100
SCALE = D ** 0.5
NORM = {F32: 6 * 2.0 ** -16, BF16: 7 * 2.0 ** -8}


class Model:
    def __init__(self, dtype, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype
        self.master = {"table": torch.randn(V, D, generator=g, device="cuda") / SCALE,
                       "up": torch.randn(EXPERTS, D, 2 * F, generator=g, device="cuda") / D ** 0.5,
                       "down": torch.randn(EXPERTS, F, D, generator=g, device="cuda") / F ** 0.5}
        self.copies = {k: w.to(dtype) if dtype != F32 else w for k, w in self.master.items()}
        self.router = torch.randn(D, EXPERTS, generator=g, device="cuda").to(dtype)
        self.tokens = torch.randint(-3, V, (T,), generator=g, device="cuda")               # some are padding
        self.target = torch.randn(T, D, generator=g, device="cuda").to(dtype)             # dloss / dy

    def step(self):
        """y and every gradient of sum(target y), the routing held fixed."""
        from fastmace_b200 import checkpoints, embedding, experts, grouped
        w = self.copies
        x = embedding.embedding(self.tokens, w["table"], SCALE)
        routes = experts.route_rows(x, self.router, TOP)
        groups = grouped.group_rows(routes.experts.view(-1), EXPERTS)
        rows = x.repeat_interleave(TOP, 0)
        weight = routes.weights.view(-1, 1).to(self.dtype)
        u = grouped.grouped_linear(rows, w["up"], groups)
        h, held_u = checkpoints.gated_rows(u, hold=True)
        held_x = checkpoints.hold_rows(rows)
        y = (grouped.grouped_linear(h, w["down"], groups).float() * weight.float()).view(T, TOP, D).sum(1)
        # backward: neither u, h nor the rows are kept
        dy = (self.target.repeat_interleave(TOP, 0).float() * weight.float()).to(self.dtype)
        dh = grouped.grouped_linear_input_gradient(dy, w["down"], groups)
        du, again = checkpoints.gated_rows_gradient(held_u, dh)
        d_down = grouped.grouped_linear_weight_gradient(again, dy, groups)
        d_up = checkpoints.held_weight_gradient(held_x, du, groups)
        dx = grouped.grouped_linear_input_gradient(du, w["up"], groups).view(T, TOP, D).float().sum(1)
        order = embedding.sort_tokens(self.tokens, V)
        d_table = embedding.embedding_gradient(dx, order, V, SCALE)
        return dict(x=x, y=y, routes=routes, held_u=held_u, held_x=held_x, weight=weight, table=d_table, up=d_up, down=d_down)


def _near(a, ref, bound, what):
    off = float((a.double() - ref).norm() / ref.norm())
    assert off <= bound, (what, off)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_training_step_against_float64(dtype):
    from fastmace_b200 import checkpoints
    model = Model(dtype, 1)
    s = model.step()
    w = {k: t.double() for k, t in model.copies.items()}
    live = model.tokens >= 0
    x = torch.where(live[:, None], w["table"][model.tokens.clamp(min=0)] * SCALE, 0.0)
    _near(s["x"], x, NORM[dtype], "x")
    e, weight = s["routes"].experts.long().view(-1), s["weight"].double()
    # forward from the rows as they are
    rows = s["x"].double().repeat_interleave(TOP, 0)
    u = torch.bmm(rows[:, None], w["up"][e])[:, 0]
    a, b = u.chunk(2, 1)
    h = a / (1 + torch.exp(-a)) * b
    y = (torch.bmm(h[:, None], w["down"][e])[:, 0] * weight).view(T, TOP, D).sum(1)
    _near(s["y"], y, NORM[dtype], "y")
    # backward from what is held
    held_x, held_u = checkpoints.release_rows(s["held_x"]).double(), checkpoints.release_rows(s["held_u"]).double()
    a, b = held_u.chunk(2, 1)
    sigma = 1 / (1 + torch.exp(-a))
    dy = model.target.double().repeat_interleave(TOP, 0) * weight
    dh = torch.bmm(w["down"][e], dy[:, :, None])[:, :, 0]
    du = torch.cat([dh * b * sigma * (1 + a * (1 - sigma)), dh * a * sigma], 1)
    d_down, d_up = torch.zeros_like(w["down"]), torch.zeros_like(w["up"])
    d_down.index_put_((e,), (a * sigma * b)[:, :, None] * dy[:, None], accumulate=True)
    d_up.index_put_((e,), held_x[:, :, None] * du[:, None], accumulate=True)
    dx = torch.bmm(w["up"][e], du[:, :, None])[:, :, 0].view(T, TOP, D).sum(1)
    d_table = torch.zeros(V, D, dtype=torch.float64, device="cuda").index_add_(0, model.tokens[live], dx[live]) * SCALE
    for name, ref in (("down", d_down), ("up", d_up), ("table", d_table)):
        _near(s[name], ref, NORM[dtype], name)
    # 8 bits themselves: a sixteenth of a value at most, and less of sums of them
    true_up = torch.zeros_like(d_up)
    a, b = u.chunk(2, 1)
    sigma = 1 / (1 + torch.exp(-a))
    true_up.index_put_((e,), rows[:, :, None] * torch.cat([dh * b * sigma * (1 + a * (1 - sigma)), dh * a * sigma], 1)[:, None], accumulate=True)
    _near(s["up"], true_up, 3 * 2.0 ** -4 + NORM[dtype], "up, of rows that are not held")


def test_gradients_against_differences():
    """Without 8 bits: float32, the gate's gradient from its rows themselves; the loss in float64 by the definition."""
    from fastmace_b200 import checkpoints, embedding, grouped
    model = Model(F32, 2)
    s = model.step()
    w, routes = model.copies, s["routes"]
    groups = grouped.group_rows(routes.experts.view(-1), EXPERTS)
    rows, dy = s["x"].repeat_interleave(TOP, 0), model.target.repeat_interleave(TOP, 0) * s["weight"]
    u = grouped.grouped_linear(rows, w["up"], groups)
    du, h = checkpoints.gated_rows_gradient(u, grouped.grouped_linear_input_gradient(dy, w["down"], groups))
    dx = grouped.grouped_linear_input_gradient(du, w["up"], groups).view(T, TOP, D).sum(1)
    grads = {"down": grouped.grouped_linear_weight_gradient(h, dy, groups), "up": grouped.grouped_linear_weight_gradient(rows, du, groups),
             "table": embedding.embedding_gradient(dx, embedding.sort_tokens(model.tokens, V), V, SCALE)}
    e, live = routes.experts.long().view(-1), model.tokens >= 0

    def loss(weights):
        x = torch.where(live[:, None], weights["table"][model.tokens.clamp(min=0)] * SCALE, 0.0).repeat_interleave(TOP, 0)
        a, b = torch.bmm(x[:, None], weights["up"][e])[:, 0].chunk(2, 1)
        return float((torch.bmm((a / (1 + torch.exp(-a)) * b)[:, None], weights["down"][e])[:, 0] * s["weight"].double()).view(T, TOP, D).sum(1).mul(model.target.double()).sum())

    g = torch.Generator(device="cuda").manual_seed(5)
    for name in grads:
        base = {k: t.double() for k, t in w.items()}
        step = torch.randn(w[name].shape, generator=g, device="cuda", dtype=torch.float64)
        t = 1e-5
        slope = (loss({**base, name: base[name] + t * step}) - loss({**base, name: base[name] - t * step})) / (2 * t)
        along = float((grads[name].double() * step).sum())
        # t^2 of the third derivative and 2^-53 / t of the loss are far below the float32 products' share
        assert abs(slope - along) <= 6 * 2.0 ** -16 * float(grads[name].double().norm() * step.norm()), (name, slope, along)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_call_gives_what_the_grouped_products_give(dtype):
    from fastmace_b200 import experts, grouped
    model = Model(dtype, 3)
    s = model.step()
    y = experts.expert_layer(s["x"], model.copies["up"], model.copies["down"], s["routes"])
    _near(y, s["y"].double(), NORM[dtype], "y")
    grouped.check_status()


def test_a_captured_step_with_adamw():
    """Forward, backward and the step of the weights in one graph: the bits of the same work without one."""
    from fastmace_b200 import grouped
    from fastmace_b200.optimiser import AdamW
    names = ("table", "up", "down")

    def make():
        model = Model(BF16, 4)
        optimiser = AdamW([model.master[k] for k in names], lr=1e-2, state_bits=8, copies=[model.copies[k] for k in names])
        return model, lambda: optimiser.step([s[k] for s in (model.step(),) for k in names])

    eager, step = make()
    for _ in range(4):
        step()
    captured, step = make()
    step()                                                   # one call of each kind outside a capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for k in names:
        assert torch.equal(eager.master[k], captured.master[k]) and torch.equal(eager.copies[k], captured.copies[k])
        assert not torch.equal(captured.master[k], Model(BF16, 4).master[k])
    grouped.check_status()


def test_launches_that_come_early_read_what_was_written_before():
    """Calls one behind the other, each on what the kernels right before it have written, without a wait in between."""
    from fastmace_b200 import embedding, experts
    g = torch.Generator(device="cuda").manual_seed(7)
    model = Model(BF16, 6)
    rounds = [(torch.randint(-3, V, (9000,), generator=g, device="cuda"), torch.randn(9000, 40, generator=g, device="cuda"),
               torch.randn(30, D, generator=g, device="cuda").to(BF16)) for _ in range(12)]
    big = torch.randn(2048, 2048, device="cuda")

    def one(tokens, dy, x, wait):
        busy = big @ big                                    # so that the launches behind it queue up
        t, d, rows = tokens.clone(), dy * 2.0, x.roll(1, 0).clone()
        if wait:
            torch.cuda.synchronize()
        grad = embedding.embedding_gradient(d, embedding.sort_tokens(t, V), V)
        few = embedding.embedding_gradient(d[:500], embedding.sort_tokens(t[:500], V), V)
        routes = experts.route_rows(rows, model.router, TOP)
        y = experts.expert_layer(rows, model.copies["up"], model.copies["down"], routes)
        t.fill_(0), d.zero_(), rows.zero_()                 # what comes behind does not come too early
        return grad, few, y, routes.weights, busy

    want = [one(*r, True) for r in rounds]
    torch.cuda.synchronize()
    got = [one(*r, False) for r in rounds]
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))


def test_captured_behind_copies_and_other_streams():
    """In a graph the launch before is not always a kernel, nor is there always just one."""
    from fastmace_b200 import embedding, experts, grouped
    model = Model(F32, 8)
    tokens, x = torch.empty_like(model.tokens), torch.empty(20, D, device="cuda")
    table = torch.empty_like(model.master["table"])
    g = torch.Generator(device="cuda").manual_seed(9)
    sources = [(torch.randint(-3, V, (T,), generator=g, device="cuda"), torch.randn(20, D, generator=g, device="cuda"), torch.randn(V, D, generator=g, device="cuda"))
               for _ in range(3)]
    now = [t.clone() for t in sources[0]]
    dy = model.target

    def work(other):
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            x.copy_(now[1])
            routes = experts.route_rows(x, model.router, TOP)
        tokens.copy_(now[0])                                # a copy of memory right before
        order = embedding.sort_tokens(tokens, V)
        table.copy_(now[2])
        torch.cuda.current_stream().wait_stream(other)
        y = experts.expert_layer(x, model.copies["up"], model.copies["down"], routes)
        return embedding.embedding(tokens, table, 2.0), embedding.embedding_gradient(dy, order, V), y

    other, side = torch.cuda.Stream(), torch.cuda.Stream()
    work(other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            got = work(other)
    for source in sources:
        for a, b in zip(now, source):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        want = work(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))
    grouped.check_status()
