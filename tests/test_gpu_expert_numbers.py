"""What the expert layer keeps of its numbers.

Between the products h = silu(a) b is a float32. The tests' a are 64, where silu(a) = a in float32, and their b are sums of powers of two that
float32 holds, so h is exact; a column of the second matrix takes one h less another, so y is their difference: each of the two is
off by half a step of 24 bits at most, their difference by one step of 23 bits more (tf32 pairs cut the last bit), and y is rounded once.
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
    assert bool(((y - want).abs() <= 2 * h * 1.01 * 2.0 ** -23 + torch.finfo(dtype).eps / 2 * want).all()), (float(y.min()), float(y.max()))
