"""Embedding rows with their gradient, the expert layer for a few tokens, and rows held in 8 bits between the forward and the
backward pass, as a program that trains or serves a model of such layers has them done.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before the
call, ``run`` is one pass, ``work`` what a pass cannot do without, ``exact`` the same from the definition in 64 bits.

Operators, by a case's ``op``:

* ``lookup``           y[r] = scale E[t(r)], zeros for a row whose token is no row of the table;
* ``lookup_gradient``  dE[v] = scale times the sum of dy[r] over the rows of token v, in fp32: the tokens sorted, then summed;
* ``experts``          the routing of a few tokens and their experts: l = x R, the ``top`` largest of softmax(l) as weights that add up
                       to one, y = sum of weight (silu(x Wg) * (x Wu)) Wd over the chosen experts;
* ``hold``             rows as e4m3 numbers with a power of two per 32 columns, exact when read back in the rows' own type; with ``gate``
                       the rows are u = (a | b), the two halves are held and h = silu(a) * b comes with them;
* ``gate_gradient``    from held u and dh: du = (da | db), and h anew;
* ``held_gradient``    dW[g] = sum over the rows of g of x[r]^T dy[r] in fp32, x held in 8 bits.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 32                                   # columns that share a power of two where rows are held in 8 bits
LOWEST = {"fp32": -117, "bf16": -117, "fp16": -15}      # of the powers; the highest, where codes end at 240 and not at 448:
HIGHEST = {"fp32": 120, "bf16": 120, "fp16": 8}


# ------------------------------------------------------------------------------------------------ the cases


def listed():
    return [
        # element embedding of the benchmark cell's atoms
        {"name": "lookup_1944_fp32", "op": "lookup", "rows": 1944, "vocabulary": 89, "width": 128, "type": "fp32", "out": "fp32",
         "scale": 1.0, "skew": 0.0, "absent": 0.0},
        # tokens of a training batch: fp32 weights, bf16 rows, scaled by the root of the width
        {"name": "lookup_65536_bf16", "op": "lookup", "rows": 65_536, "vocabulary": 100_003, "width": 2048, "type": "fp32",
         "out": "bf16", "scale": math.sqrt(2048.0), "skew": 1.05, "absent": 0.02},
        # element embedding of the large benchmark's atoms: very long sums, most of the table's rows without any
        {"name": "dlookup_884736_fp32", "op": "lookup_gradient", "rows": 884_736, "vocabulary": 89, "width": 128, "type": "fp32",
         "scale": 1.0, "skew": 2.5, "absent": 0.0},
        # tokens of a training batch: a few words in thousands of places, most of the table untouched
        {"name": "dlookup_65536_bf16", "op": "lookup_gradient", "rows": 65_536, "vocabulary": 100_003, "width": 1024, "type": "bf16",
         "scale": 32.0, "skew": 1.05, "absent": 0.02},
        # one token being decoded
        {"name": "experts_1_bf16", "op": "experts", "rows": 1, "experts": 64, "top": 8, "width": 2048, "inner": 1024, "type": "bf16"},
        # a few sequences at once, odd sizes: rows of weights at no multiple of 16 bytes
        {"name": "experts_33_odd_fp16", "op": "experts", "rows": 33, "experts": 40, "top": 3, "width": 1001, "inner": 515, "type": "fp16"},
        # a full decoding batch: every expert is read, for about eight rows
        {"name": "experts_64_bf16", "op": "experts", "rows": 64, "experts": 32, "top": 4, "width": 4096, "inner": 2048, "type": "bf16"},
        # the gate of an expert layer in a training step, its input kept in 8 bits
        {"name": "gate_16384_bf16", "op": "hold", "gate": True, "rows": 16_384, "columns": 2048, "type": "bf16"},
        # input rows of an odd-sized linear
        {"name": "hold_5003_odd_fp16", "op": "hold", "gate": False, "rows": 5003, "columns": 515, "type": "fp16"},
        # the gate's backward pass
        {"name": "dgate_16384_bf16", "op": "gate_gradient", "rows": 16_384, "columns": 2048, "type": "bf16"},
        # weight gradient of the species skip from held features, 10,368 atoms
        {"name": "dheld_10368_fp32", "op": "held_gradient", "rows": 10_368, "groups": 3, "k": 128, "n": 128, "type": "fp32",
         "skew": 0.5, "absent": 0.0},
        # weight gradient of an expert layer, training batch
        {"name": "dheld_16384_bf16", "op": "held_gradient", "rows": 16_384, "groups": 32, "k": 2048, "n": 1024, "type": "bf16",
         "skew": 0.6, "absent": 0.03},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_gradient", "lookup_gradient", "experts", "experts", "hold", "gate_gradient", "held_gradient"])
    kind = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("lookup", "lookup_gradient"):
        width = rng.choice([128, 64, 256, 512, 1024, 2048, 4096, _log(rng, 1, 2500)])
        vocabulary = min(_log(rng, 1, 200_000), 110_000_000 // width)
        case = {"op": op, "rows": max(1, min(_log(rng, 1, 900_000), 130_000_000 // width)), "vocabulary": vocabulary, "width": width,
                "type": kind, "scale": rng.choice([1.0, math.sqrt(width)]), "skew": rng.choice([0.0, 1.05, 2.0]),
                "absent": rng.choice([0.0, 0.02, 0.5])}
        if op == "lookup":
            case["out"] = rng.choice([kind, "fp32", "bf16"])
        return case
    if op == "experts":
        width, inner = (rng.choice([128, 512, 1024, 2048, 4096, _log(rng, 16, 2500)]) for _ in range(2))
        experts = _log(rng, 1, 256)
        while experts * width * inner > (100_000_000 if kind == "fp32" else 200_000_000):
            experts = max(1, experts // 2)
        rows = _log(rng, 1, 64)
        return {"op": op, "rows": rows, "experts": experts, "top": rng.randint(1, min(8, experts)), "width": width, "inner": inner,
                "type": kind}
    if op == "held_gradient":
        groups, rows = _log(rng, 1, 256), _log(rng, 1, 400_000)
        k, n = (rng.choice([128, 64, 256, 512, 1024, 2048, 4096, _log(rng, 16, 2500)]) for _ in range(2))
        while groups * k * n > 100_000_000:
            groups = groups // 2
        most = (1e10 if kind == "fp32" else 3e10) / (k * n)
        return {"op": op, "rows": max(1, min(rows, int(most), 100_000_000 // (k + n))), "groups": groups, "k": k, "n": n, "type": kind,
                "skew": rng.choice([0.0, 0.4, 0.8]), "absent": rng.choice([0.0, 0.05])}
    columns = rng.choice([128, 256, 512, 1024, 2048, 4096, 2 * _log(rng, 1, 2500)])
    rows = max(1, min(_log(rng, 1, 200_000), 60_000_000 // columns))
    case = {"op": op, "rows": rows, "columns": columns, "type": kind}
    if op == "hold":
        case["gate"] = rng.choice([True, False])
    return case


# ------------------------------------------------------------------------------------------------ inputs


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _drawn(weight, count, g):
    """Numbers drawn with these weights; the running sum is made on the host, where its order is always the same."""
    sums = weight.cpu().cumsum(0).cuda()
    at = torch.rand(count, dtype=torch.float64, generator=g, device="cuda") * sums[-1]
    return torch.searchsorted(sums, at, right=True).clamp(max=len(weight) - 1)


def _tokens(case, g):
    """Token numbers whose frequencies fall with a power of their rank, the ranks dealt to the table's rows at random."""
    size = case["vocabulary"]
    rank = _drawn((torch.arange(size, dtype=torch.float64) + 2.7) ** -case["skew"], case["rows"], g)
    tokens = torch.randperm(size, generator=g, device="cuda")[rank].to(torch.int32)
    gone = torch.rand(case["rows"], generator=g, device="cuda") < case["absent"]
    return torch.where(gone, torch.full_like(tokens, -1), tokens)


def _activations(g, rows, columns, kind):
    """Rows whose columns differ in size, with a few values far above the others, as activations have them."""
    x = _randn(g, rows, columns) * torch.exp(0.5 * _randn(g, columns))
    return (x * torch.where(torch.rand(rows, columns, generator=g, device="cuda") < 1e-3, 20.0, 1.0)).to(TYPES[kind])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    op, kind = case["op"], TYPES.get(case["type"])
    if op in ("lookup", "lookup_gradient"):
        s["tokens"] = _tokens(case, g)
        if op == "lookup":
            s["table"] = (_randn(g, case["vocabulary"], case["width"]) * 0.02).to(kind)
        else:
            s["dy"] = _randn(g, case["rows"], case["width"]).mul_(1e-2).to(kind)
        return s
    if op == "experts":
        t, e, d, f = case["rows"], case["experts"], case["width"], case["inner"]
        s["x"] = _randn(g, t, d).to(kind)
        s["router"] = (_randn(g, d, e) * (1.5 / math.sqrt(d))).to(kind)
        s["w_up"] = _randn(g, e, d, 2 * f).mul_(1.0 / math.sqrt(d)).to(kind)      # gate columns, then those they multiply
        s["w_down"] = _randn(g, e, f, d).mul_(1.0 / math.sqrt(f)).to(kind)
        return s
    if op == "held_gradient":
        keys = _drawn(torch.exp(case["skew"] * _randn(g, case["groups"])).double(), case["rows"], g)
        gone = torch.rand(case["rows"], generator=g, device="cuda") < case["absent"]
        group = torch.where(gone, torch.full_like(keys, case["groups"]), keys)
        s["rows"] = torch.sort(group, stable=True).indices.to(torch.int32)
        count = torch.bincount(group, minlength=case["groups"] + 1)[:case["groups"]]
        s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
        s["most"] = int(count.max())              # rows of the largest group, for the plain form's padded arrays
        s["dy"] = _randn(g, case["rows"], case["n"]).mul_(1e-2).to(kind)
        s["codes"], s["exponents"] = _plain_hold(_activations(g, case["rows"], case["k"], case["type"]), case["type"])
        return s
    x = _activations(g, case["rows"], case["columns"], case["type"])
    if op == "hold":
        s["x"] = x
        return s
    half = case["columns"] // 2
    held = [_plain_hold(part, case["type"]) for part in (x[:, :half], x[:, half:])]
    s["codes"], s["exponents"] = (torch.cat(parts, 1) for parts in zip(*held))
    s["dh"] = _randn(g, case["rows"], half).mul_(1e-2).to(kind)
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _padded_columns(x):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).reshape(x.shape[0], -1, BLOCK)


def _plain_hold(x, kind):
    """Codes [rows, columns] in e4m3 and, per 32 columns, the exponent of their unit, plus 127 (uint8)."""
    blocks = _padded_columns(x.float())
    mantissa, power = torch.frexp(blocks.abs().amax(2))              # the largest = mantissa 2^power, 0.5 <= mantissa < 1
    e = power - 9 + (mantissa > 0.875).to(torch.int32)               # 448 = 0.875 x 2^9
    e = e.clamp(LOWEST[kind], HIGHEST[kind])
    most = torch.where(e == HIGHEST[kind], 240.0, 448.0)[:, :, None]
    unit = torch.ldexp(blocks, -e[:, :, None])
    codes = torch.minimum(torch.maximum(unit, -most), most).to(torch.float8_e4m3fn)
    return codes.reshape(x.shape[0], -1)[:, :x.shape[1]].contiguous(), (e + 127).to(torch.uint8)


def _released(codes, exponents):
    unit = torch.ldexp(torch.ones((), device="cuda"), exponents.to(torch.int32) - 127)
    return (_padded_columns(codes.float()) * unit[:, :, None]).reshape(len(codes), -1)[:, :codes.shape[1]]


def _halves(s):
    half, blocks = s["case"]["columns"] // 2, s["exponents"].shape[1] // 2
    return (_released(s["codes"][:, :half], s["exponents"][:, :blocks]), _released(s["codes"][:, half:], s["exponents"][:, blocks:]))


def _plain_lookup(s):
    case, tokens = s["case"], s["tokens"].long()
    there = (tokens >= 0) & (tokens < case["vocabulary"])
    row = s["table"][tokens.clamp(0, case["vocabulary"] - 1)].float() * case["scale"]
    return torch.where(there[:, None], row, 0.0).to(TYPES[case["out"]])


def _plain_lookup_gradient(s):
    case, tokens = s["case"], s["tokens"].long()
    size = case["vocabulary"]
    tokens = torch.where((tokens >= 0) & (tokens < size), tokens, size)
    # long sums in 64 bits
    held = torch.float64 if case["rows"] > 1000 * min(size, 100) else torch.float32
    out = torch.zeros(size + 1, case["width"], dtype=held, device="cuda").index_add_(0, tokens, s["dy"].to(held))
    return (out[:size] * case["scale"]).float()


def _plain_routes(s):
    """Logits in 64 bits, since a choice goes by their order; equal ones in the order of their numbers."""
    logits = s["x"].double() @ s["router"].double()
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :s["case"]["top"]]
    return order, torch.softmax(torch.gather(logits, 1, order), 1).float()


def _plain_experts(s):
    case = s["case"]
    t, top, f = case["rows"], case["top"], case["inner"]
    chosen, weight = _plain_routes(s)
    if t * top < case["experts"]:
        # the matrices of each pair of token and expert
        x = s["x"].float().repeat_interleave(top, 0)[:, None]
        u = torch.bmm(x, s["w_up"][chosen.reshape(-1)].float())
        h = u[:, :, :f] * torch.sigmoid(u[:, :, :f]) * u[:, :, f:]
        y = torch.bmm(h, s["w_down"][chosen.reshape(-1)].float()).view(t, top, -1)
        y = (y * weight[:, :, None]).sum(1)
    else:
        # every expert for every token, weighted with zero where it is not chosen
        scale = torch.zeros(t, case["experts"], device="cuda").scatter_(1, chosen, weight)
        u = torch.matmul(s["x"].float(), s["w_up"].float())
        h = u[:, :, :f] * torch.sigmoid(u[:, :, :f]) * u[:, :, f:]
        y = (torch.bmm(h, s["w_down"].float()) * scale.t()[:, :, None]).sum(0)
    return {"y": y.to(s["x"].dtype), "experts": chosen.to(torch.int32), "weights": weight}


def _plain_hold_case(s):
    case = s["case"]
    if not case["gate"]:
        return _plain_hold(s["x"], case["type"])
    half = case["columns"] // 2
    a, b = s["x"][:, :half], s["x"][:, half:]
    h = (a.float() * torch.sigmoid(a.float()) * b.float()).to(s["x"].dtype)
    held = [_plain_hold(part, case["type"]) for part in (a, b)]
    return (h, *(torch.cat(parts, 1) for parts in zip(*held)))


def _plain_gate_gradient(s):
    (a, b), dh = _halves(s), s["dh"].float()
    sigma = torch.sigmoid(a)
    da = dh * b * sigma * (1.0 + a * (1.0 - sigma))
    db = dh * a * sigma
    return torch.cat([da, db], 1).to(s["dh"].dtype), (a * sigma * b).to(s["dh"].dtype)


def _plain_held_gradient(s):
    chunk = 4096                                   # long sums by chunks, and the chunks' sums in 64 bits
    most = max(1, s["most"])
    most = most if most <= chunk else -(-most // chunk) * chunk
    at = s["offsets"][:-1, None].long() + torch.arange(most, device="cuda")
    live = at < s["offsets"][1:, None]
    row = s["rows"].long()[at.clamp(max=len(s["rows"]) - 1)]
    x = _released(s["codes"], s["exponents"])
    a, b = (torch.where(live[:, :, None], t[row], 0.0) for t in (x, s["dy"].float()))
    groups, parts = a.shape[0], max(1, most // chunk)
    a, b = (t.reshape(groups * parts, most // parts, t.shape[2]) for t in (a, b))
    part = torch.bmm(a.transpose(1, 2), b).reshape(groups, parts, a.shape[2], b.shape[2])
    return part[:, 0] if parts == 1 else part.sum(1, dtype=torch.float64).float()


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    op, case = s["case"]["op"], s["case"]
    if own:
        from fastmace_b200 import checkpoints, embedding, experts, grouped

        if op == "lookup":
            return embedding.embedding(s["tokens"], s["table"], case["scale"], dtype=TYPES[case["out"]])
        if op == "lookup_gradient":
            order = embedding.sort_tokens(s["tokens"], case["vocabulary"])
            return embedding.embedding_gradient(s["dy"], order, case["vocabulary"], case["scale"])
        if op == "experts":
            routes = experts.route_rows(s["x"], s["router"], case["top"])
            y = experts.expert_layer(s["x"], s["w_up"], s["w_down"], routes)
            return {"y": y, "experts": routes.experts, "weights": routes.weights}
        if op == "hold":
            if case["gate"]:
                h, held = checkpoints.gated_rows(s["x"], hold=True)
                return h, held.codes, held.exponents
            held = checkpoints.hold_rows(s["x"])
            return held.codes, held.exponents
        if op == "gate_gradient":
            held = checkpoints.HeldRows(s["codes"], s["exponents"], s["dh"].dtype, parts=2)
            return checkpoints.gated_rows_gradient(held, s["dh"])
        held = checkpoints.HeldRows(s["codes"], s["exponents"], s["dy"].dtype)
        return checkpoints.held_weight_gradient(held, s["dy"], grouped.RowGroups(s["rows"], s["offsets"]))
    return {"lookup": _plain_lookup, "lookup_gradient": _plain_lookup_gradient, "experts": _plain_experts, "hold": _plain_hold_case,
            "gate_gradient": _plain_gate_gradient, "held_gradient": _plain_held_gradient}[op](s)


def _distinct(case):
    """Rows of the table that the tokens of a case name, on average."""
    weight = [(i + 2.7) ** -case["skew"] for i in range(case["vocabulary"])]
    total, rows = sum(weight), case["rows"] * (1.0 - case["absent"])
    return sum(-math.expm1(rows * math.log1p(-w / total)) if w < total else min(1.0, rows) for w in weight)


def work(case):
    op, rows, e = case["op"], case["rows"], BYTES[case["type"]]
    if op == "lookup":
        return {"bytes": 4 * rows + case["width"] * (_distinct(case) * e + rows * BYTES[case["out"]]), "flops": rows * case["width"]}
    if op == "lookup_gradient":
        live = rows * (1.0 - case["absent"])
        return {"bytes": 4 * rows + case["width"] * (live * e + 4 * case["vocabulary"]), "flops": live * case["width"]}
    if op == "experts":
        touched = case["experts"] * -math.expm1(rows * math.log1p(-case["top"] / case["experts"])) if case["top"] < case["experts"] \
            else case["experts"]
        d, f = case["width"], case["inner"]
        return {"bytes": e * (3 * touched * d * f + 2 * rows * d + d * case["experts"]) + 8 * rows * case["top"],
                "flops": 2.0 * rows * (3 * case["top"] * d * f + d * case["experts"])}
    if op == "held_gradient":
        m = rows * (1.0 - case["absent"])
        return {"bytes": m * (case["k"] * (1 + 1 / BLOCK) + e * case["n"] + 4) + 4 * case["groups"] * case["k"] * case["n"],
                "flops": 2.0 * m * case["k"] * case["n"]}
    values = rows * case["columns"]
    if op == "hold":
        return {"bytes": values * (e + 1 + 1 / BLOCK + (e / 2 if case["gate"] else 0)), "flops": (8 if case["gate"] else 4) * values}
    return {"bytes": values * (1 + 1 / BLOCK + e / 2 + e + e / 2), "flops": 8 * values}


# ------------------------------------------------------------------------------------------------ in 64 bits


def _exact_e4m3(x):
    """The nearest number of four exponent and three fraction bits, ties to an even fraction: spacing 2^(e - 3) between 2^e and
    2^(e + 1), 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_hold(x, kind):
    """Codes and exponents, both from the powers of two between which the largest of 32 columns lies."""
    blocks = _padded_columns(x.double())
    largest = blocks.abs().max(2).values
    e = torch.full_like(largest, float(LOWEST[kind]))
    for power in range(LOWEST[kind] + 1, HIGHEST[kind] + 1):
        e = torch.where(largest > 448.0 * 2.0 ** (power - 1), float(power), e)
    most = torch.where(e == HIGHEST[kind], 240.0, 448.0)[:, :, None]
    codes = _exact_e4m3((blocks * torch.exp2(-e)[:, :, None]).clamp(-most, most))
    return codes.reshape(len(x), -1)[:, :x.shape[1]], (e + 127).to(torch.uint8)


def _exact_held(codes, exponents):
    power = torch.exp2(exponents.double() - 127).repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.double() * power


def _exact_silu(a):
    return a / (1.0 + torch.exp(-a))


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        tokens = s["tokens"].long()
        out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
        live = torch.nonzero((tokens >= 0) & (tokens < case["vocabulary"]))[:, 0]
        out[live] = s["table"].double()[tokens[live]] * case["scale"]
        return out
    if op == "lookup_gradient":
        # differences of the running sum of the sorted rows
        tokens, order = torch.sort(s["tokens"])
        total = torch.cat([torch.zeros(1, case["width"], dtype=torch.float64, device="cuda"), s["dy"][order].double().cumsum(0)])
        at = torch.searchsorted(tokens, torch.arange(case["vocabulary"] + 1, dtype=torch.int32, device="cuda"))
        return (total[at[1:]] - total[at[:-1]]) * case["scale"]
    if op == "experts":
        logits = s["x"].double() @ s["router"].double()
        weight, chosen = torch.topk(logits, case["top"], 1)
        weight = torch.exp(weight - weight[:, :1])
        weight = weight / weight.sum(1, keepdim=True)
        y = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
        for e in chosen.unique().tolist():
            t, j = torch.nonzero(chosen == e, as_tuple=True)
            a, b = (s["x"][t].double() @ s["w_up"][e].double()).chunk(2, 1)
            y.index_add_(0, t, (_exact_silu(a) * b) @ s["w_down"][e].double() * weight[t, j][:, None])
        return {"y": y, "experts": chosen.to(torch.int32), "weights": weight}
    if op == "hold":
        if not case["gate"]:
            return _exact_hold(s["x"], case["type"])
        a, b = s["x"].chunk(2, 1)
        held = [_exact_hold(part, case["type"]) for part in (a, b)]
        return (_exact_silu(a.double()) * b.double(), *(torch.cat(parts, 1) for parts in zip(*held)))
    if op == "gate_gradient":
        codes, exponents, dh = s["codes"].float().chunk(2, 1), s["exponents"].chunk(2, 1), s["dh"].double()
        a, b = (_exact_held(c, e) for c, e in zip(codes, exponents))
        sigma = 1.0 / (1.0 + torch.exp(-a))
        slope = sigma + a * sigma * (1.0 - sigma)
        return torch.cat([dh * b * slope, dh * _exact_silu(a)], 1), _exact_silu(a) * b
    x = _exact_held(s["codes"].float(), s["exponents"])
    out = torch.zeros(case["groups"], case["k"], case["n"], dtype=torch.float64, device="cuda")
    start = s["offsets"].tolist()
    for g, (begin, end) in enumerate(zip(start, start[1:])):
        r = s["rows"][begin:end].long()
        if end > begin:
            out[g] = x[r].t() @ s["dy"][r].double()
    return out
