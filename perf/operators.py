"""The grouped products of a species-dependent (or expert) linear with their gradients, and the AdamW step over a model's
weights, as a program that trains such weights has them done.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds before the
call, ``run`` is one pass, ``work`` what a pass cannot do without, ``exact`` the same from the definition in 64 bits.

Operators, by a case's ``op``:

* ``group``            which rows belong to which group: a stable order of the rows by key and where each group starts;
* ``linear``           y[r] = x[r] W[g(r)] for the rows of every group, zeros for rows of none;
* ``input_gradient``   dx[r] = dy[r] W[g(r)]^T;
* ``weight_gradient``  dW[g] = sum over the rows of g of x[r]^T dy[r], in fp32;
* ``adamw``            one step over a list of tensors, moments in 32 or in 8 bits, optionally with a bf16 copy of the weights.
"""

from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BLOCK = 256                  # values that share a scale where moments are held in 8 bits; every tensor starts a block
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEPS_BEFORE = 7             # steps the moments of a prepared state have seen


# ------------------------------------------------------------------------------------------------ the cases


def listed():
    return [
        # the benchmark cell's atoms by species
        {"name": "group_1944_atoms", "op": "group", "rows": 1944, "groups": 2, "skew": 0.0, "absent": 0.0},
        # tokens of a large batch by expert, a twentieth of them padding
        {"name": "group_2m_rows", "op": "group", "rows": 2_100_003, "groups": 128, "skew": 0.8, "absent": 0.05},
        # species skip of the benchmark cell: scalar part of the node features [atom][4][128]
        {"name": "skip_1944_fp32", "op": "linear", "rows": 1944, "groups": 2, "k": 128, "n": 128, "type": "fp32",
         "stride": 4, "skew": 0.0, "absent": 0.0},
        # the same layer of a five-species cell of the large benchmark's size
        {"name": "skip_884736_fp32", "op": "linear", "rows": 884_736, "groups": 5, "k": 128, "n": 128, "type": "fp32",
         "stride": 1, "skew": 0.5, "absent": 0.0},
        # eight single tokens among 64 experts: each touched matrix is read for a row or two
        {"name": "tokens_8_bf16", "op": "linear", "rows": 8, "groups": 64, "k": 2048, "n": 1024, "type": "bf16",
         "stride": 1, "skew": 0.0, "absent": 0.0},
        # a prompt's tokens over 32 experts of uneven load, some rows padding
        {"name": "prompt_16384_bf16", "op": "linear", "rows": 16_384, "groups": 32, "k": 2048, "n": 2048, "type": "bf16",
         "stride": 1, "skew": 0.6, "absent": 0.03},
        # adjoint of an odd-sized layer, half precision: 515 columns make rows of no particular alignment
        {"name": "adjoint_odd_fp16", "op": "input_gradient", "rows": 5003, "groups": 17, "k": 1000, "n": 515,
         "type": "fp16", "stride": 1, "skew": 0.8, "absent": 0.05},
        # weight gradient of the species skip, 10,368 atoms of a three-species cell
        {"name": "dskip_10368_fp32", "op": "weight_gradient", "rows": 10_368, "groups": 3, "k": 128, "n": 128,
         "type": "fp32", "stride": 4, "skew": 0.5, "absent": 0.0},
        # weight gradient of an expert layer, training batch
        {"name": "dexperts_16384_bf16", "op": "weight_gradient", "rows": 16_384, "groups": 32, "k": 2048, "n": 1024,
         "type": "bf16", "stride": 1, "skew": 0.6, "absent": 0.03},
        # the 43 tensors of the medium model
        {"name": "adamw_medium_model", "op": "adamw", "tensors": 0, "values": 4_688_400, "bits": 32, "gradient": "fp32",
         "copy": False},
        # experts of a few layers, moments in 8 bits, gradients in bf16, bf16 copy for the products
        {"name": "adamw_8bit_64m", "op": "adamw", "tensors": 150, "values": 64_000_000, "bits": 8, "gradient": "bf16",
         "copy": True},
        # a whole model of 200 M weights, moments in 32 bits
        {"name": "adamw_200m", "op": "adamw", "tensors": 290, "values": 200_000_000, "bits": 32, "gradient": "fp32",
         "copy": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["group", "linear", "linear", "input_gradient", "weight_gradient", "weight_gradient", "adamw"])
    if op == "group":
        return {"op": op, "rows": _log(rng, 1, 2_100_000), "groups": _log(rng, 1, 1024), "skew": rng.choice([0.0, 0.8]),
                "absent": rng.choice([0.0, 0.05, 0.5])}
    if op == "adamw":
        return {"op": op, "tensors": _log(rng, 1, 300), "values": _log(rng, 10_000, 100_000_000), "bits": rng.choice([8, 32]),
                "gradient": rng.choice(["fp32", "bf16", "fp16"]), "copy": rng.choice([True, False])}
    kind = rng.choice(["fp32", "bf16", "fp16"])
    groups, rows = _log(rng, 1, 256), _log(rng, 1, 400_000)
    # species layers have 128 channels, expert layers up to 4096; a third of the sizes are odd
    k, n = (rng.choice([128, 64, 256, 512, 1024, 2048, 4096, _log(rng, 16, 2500)]) for _ in range(2))
    while groups * k * n > 150_000_000:
        groups = groups // 2
    most = (2e10 if kind == "fp32" else 6e10) / (k * n)
    rows = max(1, min(rows, int(most), 120_000_000 // (k + n)))
    return {"op": op, "rows": rows, "groups": groups, "k": k, "n": n, "type": kind, "stride": rng.choice([1, 1, 4]),
            "skew": rng.choice([0.0, 0.4, 0.8]), "absent": rng.choice([0.0, 0.0, 0.05])}


def model_sizes():
    """Values of each tensor of the medium model's weights (two interactions, 128 channels, 89 elements)."""
    c, z = 128, 89
    first = [c * c] + [8 * 64, 64 * 64, 64 * 64, 64 * 4 * c] + [c * c] * 4 + [c * z * c]
    first += [z * 1 * c, z * 4 * c, z * 23 * c, c * c, z * 1 * c, z * 6 * c, z * 51 * c, c * c, c]
    second = [c * c] * 2 + [8 * 64, 64 * 64, 64 * 64, 64 * 10 * c] + [c * c] * 10 + [c * z * c]
    second += [z * 1 * c, z * 4 * c, z * 23 * c, c * c, c * 16, 16]
    return [z * c] + first + second


def tensor_sizes(case):
    """Values of each tensor of an ``adamw`` case: the medium model's, or sizes that differ by up to a factor of a hundred and
    add up to about ``values``, the same for every seed of the inputs."""
    if not case["tensors"]:
        return model_sizes()
    rng = random.Random(case["values"])
    shares = [math.exp(rng.uniform(0.0, math.log(100.0))) for _ in range(case["tensors"])]
    return [max(1, int(case["values"] * s / sum(shares))) for s in shares]


# ------------------------------------------------------------------------------------------------ inputs


def _keys(case, g):
    groups = case["groups"]
    weight = torch.exp(case["skew"] * torch.randn(groups, generator=g, device="cuda"))
    keys = torch.multinomial(weight, case["rows"], replacement=True, generator=g).to(torch.int32)
    if case["absent"] > 0:
        gone = torch.rand(case["rows"], generator=g, device="cuda") < case["absent"]
        keys = torch.where(gone, torch.full_like(keys, -1), keys)
    return keys


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _strided(g, rows, width, stride, kind):
    """[rows, width] of a wider array [rows, stride, width], as one component of the node features is."""
    return _randn(g, rows, stride, width).to(TYPES[kind])[:, 0, :]


def _e4m3(x):
    return x.to(torch.float8_e4m3fn)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "adamw":
        sizes = tensor_sizes(case)
        padded = [-(-n // BLOCK) * BLOCK for n in sizes]
        starts = [0]
        for n in padded:
            starts.append(starts[-1] + n)
        total = starts[-1]
        live = torch.zeros(total, dtype=torch.bool, device="cuda")
        for n, at in zip(sizes, starts):
            live[at:at + n] = True
        # weights and gradients of a program that keeps each in one buffer, every tensor at the start of a block
        p, grad, m = (_randn(g, total).mul_(live) for _ in range(3))
        r = _randn(g, total).abs_().mul_(live)
        # gradients of layers differ by orders of magnitude
        size = torch.exp(2.0 * _randn(g, total // BLOCK)).repeat_interleave(BLOCK)
        p, grad, m, r = p * 0.05, (grad * size * 1e-3).to(TYPES[case["gradient"]]), m * size * 3e-4, (r + 0.1 * live) * size * 1e-3
        s.update(p=p, grad=grad, step=STEPS_BEFORE)
        if case["copy"]:
            s["copy"] = torch.zeros(total, dtype=torch.bfloat16, device="cuda")
        if case["bits"] == 8:
            for name, x in (("m", m), ("r", r)):
                scale = (x.view(-1, BLOCK).abs().amax(1) / 448.0).clamp(min=2.0 ** -126)
                s[name], s[name + "_scale"] = _e4m3(x.view(-1, BLOCK) / scale[:, None]).view(-1), scale
        else:
            s.update(m=m, v=r * r)
        if own:
            from fastmace_b200.optimiser import AdamW

            cut = lambda x: [x[at:at + n] for n, at in zip(sizes, starts)]  # noqa: E731
            s["optimiser"] = AdamW(cut(p), lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=case["bits"],
                                   copies=cut(s["copy"]) if case["copy"] else None)
            moments = (s["m"], s["m_scale"], s["r"], s["r_scale"]) if case["bits"] == 8 else (s["m"], s["v"])
            s["optimiser"].load_moments(STEPS_BEFORE, *moments)
            s["grads"] = cut(grad)
        return s
    keys = _keys(case, g)
    if case["op"] == "group":
        s["keys"] = keys
        return s
    group = torch.where((keys < 0) | (keys >= case["groups"]), torch.full_like(keys, case["groups"]), keys)
    s["rows"] = torch.sort(group, stable=True).indices.to(torch.int32)
    count = torch.bincount(group, minlength=case["groups"] + 1)[:case["groups"]]
    s["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
    s["most"] = int(count.max())              # rows of the largest group, for the plain form's padded arrays
    m, k, n, kind = case["rows"], case["k"], case["n"], case["type"]
    if case["op"] != "input_gradient":
        s["x"] = _strided(g, m, k, case["stride"], kind)
    if case["op"] != "linear":
        s["dy"] = _strided(g, m, n, case["stride"] if case["op"] == "input_gradient" else 1, kind)
    if case["op"] != "weight_gradient":
        s["w"] = (_randn(g, case["groups"], k, n) / math.sqrt(k if case["op"] == "linear" else n)).to(TYPES[kind])
    return s


# ------------------------------------------------------------------------------------------------ plain forms


def _padded(s, most):
    """Row numbers of every group side by side, [groups, most], and which of them are rows of the group."""
    at = s["offsets"][:-1, None].long() + torch.arange(most, device="cuda")
    live = at < s["offsets"][1:, None]
    return s["rows"].long()[at.clamp(max=len(s["rows"]) - 1)], live


def _plain_group(s):
    groups = s["case"]["groups"]
    keys = s["keys"].long()
    key = torch.where((keys < 0) | (keys >= groups), torch.full_like(keys, groups), keys)
    order = torch.sort(key, stable=True).indices
    starts = torch.searchsorted(key[order], torch.arange(groups + 1, device="cuda"))
    return order.to(torch.int32), starts.to(torch.int32)


def _plain_product(s, a, w):
    m = a.shape[0]
    row, live = _padded(s, max(1, s["most"]))
    y = torch.bmm(torch.where(live[:, :, None], a[row].float(), 0.0), w.float())
    out = torch.zeros(m + 1, y.shape[2], device="cuda")
    out[torch.where(live, row, m)] = y            # what is no row of the group goes to a row that is dropped
    return out[:m].to(a.dtype)


def _plain_weight_gradient(s):
    chunk = 4096                                   # long sums by chunks, and the chunks' sums in 64 bits
    most = max(1, s["most"])
    most = most if most <= chunk else -(-most // chunk) * chunk
    row, live = _padded(s, most)
    a, b = (torch.where(live[:, :, None], t[row].float(), 0.0) for t in (s["x"], s["dy"]))
    groups, parts = a.shape[0], max(1, most // chunk)
    a, b = (t.view(groups * parts, most // parts, t.shape[2]) for t in (a, b))
    part = torch.bmm(a.transpose(1, 2), b).view(groups, parts, a.shape[2], b.shape[2])
    return part[:, 0] if parts == 1 else part.sum(1, dtype=torch.float64).float()


def _plain_adamw(s):
    eight = s["case"]["bits"] == 8
    s["step"] += 1
    t, p, grad = s["step"], s["p"], s["grad"].float()
    if eight:
        m = s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]
        r = s["r"].float().view(-1, BLOCK) * s["r_scale"][:, None]
        m, v = m.view(-1), (r * r).view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m * BETA1 + grad * (1.0 - BETA1)
    v = v * BETA2 + grad * (1.0 - BETA2) * grad
    root = v.sqrt()
    p.mul_(1.0 - LR * DECAY).sub_(m * (LR / (1.0 - BETA1 ** t)) / (root * (1.0 / math.sqrt(1.0 - BETA2 ** t)) + EPS))
    if s["case"]["copy"]:
        s["copy"].copy_(p)
    if eight:
        for name, x in (("m", m), ("r", root)):
            x = x.view(-1, BLOCK)
            scale = (x.abs().amax(1) / 448.0).clamp(min=2.0 ** -126)
            code = _e4m3(x / scale[:, None])
            if name == "r":                        # a second moment that is not zero is never held as zero
                code = torch.where((x > 0) & (code.float() == 0), torch.full_like(x, 2.0 ** -9), code.float()).to(code.dtype)
            s[name].copy_(code.view(-1))
            s[name + "_scale"].copy_(scale)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)


def _adamw_state(s):
    """The step's outputs: weights, their copy and the moments. Moments in 8 bits come as the numbers held (e4m3, in units of
    their block's scale) and the scales."""
    names = ("p", "copy", "m", "r", "m_scale", "r_scale") if s["case"]["bits"] == 8 else ("p", "copy", "m", "v")
    return {name: s[name] for name in names if name in s}


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    op = s["case"]["op"]
    if own:
        from fastmace_b200 import grouped

        if op == "adamw":
            s["optimiser"].step(s["grads"])
            return _adamw_state(s)
        if op == "group":
            return tuple(grouped.group_rows(s["keys"], s["case"]["groups"]))
        groups = grouped.RowGroups(s["rows"], s["offsets"])
        if op == "linear":
            return grouped.grouped_linear(s["x"], s["w"], groups)
        if op == "input_gradient":
            return grouped.grouped_linear_input_gradient(s["dy"], s["w"], groups)
        return grouped.grouped_linear_weight_gradient(s["x"], s["dy"], groups)
    if op == "adamw":
        _plain_adamw(s)
        return _adamw_state(s)
    if op == "group":
        return _plain_group(s)
    if op == "linear":
        return _plain_product(s, s["x"], s["w"])
    if op == "input_gradient":
        return _plain_product(s, s["dy"], s["w"].transpose(1, 2))
    return _plain_weight_gradient(s)


def work(case):
    if case["op"] == "group":
        return {"bytes": 8 * case["rows"] + 4 * (case["groups"] + 1), "flops": 0}
    if case["op"] == "adamw":
        total = sum(tensor_sizes(case))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": total * (8 + BYTES[case["gradient"]] + moments + (2 if case["copy"] else 0)), "flops": 16 * total}
    m, k, n, e = case["rows"] * (1.0 - case["absent"]), case["k"], case["n"], BYTES[case["type"]]
    flops = 2.0 * m * k * n
    if case["op"] == "weight_gradient":
        return {"bytes": e * m * (k + n) + 4 * case["groups"] * k * n + 4 * m, "flops": flops}
    touched = case["groups"] * -math.expm1(m * math.log1p(-1.0 / case["groups"])) if case["groups"] > 1 else 1
    wide_in, wide_out = (k, n) if case["op"] == "linear" else (n, k)
    return {"bytes": e * (m * wide_in + case["rows"] * wide_out + touched * k * n) + 4 * m, "flops": flops}


# ------------------------------------------------------------------------------------------------ in 64 bits


def _exact_e4m3(x):
    """The nearest number of four exponent and three fraction bits, ties to an even fraction: spacing 2^(e - 3) between 2^e and
    2^(e + 1), 2^-9 below 2^-6, largest 448."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    return (torch.round(x / torch.exp2(e - 3)) * torch.exp2(e - 3)).clamp(-448.0, 448.0)


def _exact_adamw(s):
    t, grad, eight = s["step"] + 1, s["grad"].double(), s["case"]["bits"] == 8
    if eight:
        m, root = (s[a].double() * s[a + "_scale"].double().repeat_interleave(BLOCK) for a in ("m", "r"))
        v = root ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = BETA1 * m + (1 - BETA1) * grad
    v = BETA2 * v + (1 - BETA2) * grad ** 2
    update = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
    p = s["p"].double()
    p = p - LR * (update + DECAY * p)
    out = {"p": p}
    if s["case"]["copy"]:
        out["copy"] = p
    if not eight:
        return {**out, "m": m, "v": v}
    for name, x in (("m", m), ("r", v ** 0.5)):
        scale = (x.view(-1, BLOCK).abs().max(1).values / 448).clamp(min=2.0 ** -126)
        unit = (x.view(-1, BLOCK) / scale[:, None]).view(-1)
        code = _exact_e4m3(unit)
        out[name] = torch.where((unit > 0) & (code == 0), 2.0 ** -9, code) if name == "r" else code
        out[name + "_scale"] = scale
    return out


def exact(case, seed):
    if case["op"] == "group":
        return None
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    start = s["offsets"].tolist()
    spans = [(g, s["rows"][a:b].long()) for g, (a, b) in enumerate(zip(start, start[1:])) if b > a]
    if case["op"] == "weight_gradient":
        out = torch.zeros(case["groups"], case["k"], case["n"], dtype=torch.float64, device="cuda")
        for g, r in spans:
            out[g] = s["x"][r].double().t() @ s["dy"][r].double()
        return out
    forward = case["op"] == "linear"
    a = s["x"] if forward else s["dy"]
    out = torch.zeros(case["rows"], case["n"] if forward else case["k"], dtype=torch.float64, device="cuda")
    for g, r in spans:
        w = s["w"][g].double()
        out[r] = a[r].double() @ (w if forward else w.t())
    return out
