"""Arms of the embedding, routing and expert kernels that other tests' sizes do not reach, against plain float64 evaluations."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _beside(t, extra, front=0):
    """The same rows, with `extra` values between them and `front` before the first."""
    out = torch.full((t.shape[0], t.shape[1] + extra), float("nan"), dtype=t.dtype, device=t.device)
    out[:, front:front + t.shape[1]] = t
    return out[:, front:front + t.shape[1]]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,vocabulary,width", [(40_000, 30, 512), (9000, 5000, 264), (200_000, 89, 128), (30_000, 7, 1024)])
def test_gradient_of_rows_has_the_same_bits_wherever_they_lie(rows, vocabulary, width, dtype):
    from fastmace_b200 import embedding
    g = torch.Generator(device="cuda").manual_seed(rows)
    order = embedding.sort_tokens(torch.randint(-1, vocabulary, (rows,), generator=g, device="cuda"), vocabulary)
    dy = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    want = embedding.embedding_gradient(dy, order, vocabulary, 3.0)
    base = torch.randn(vocabulary, width, generator=g, device="cuda")
    more = embedding.embedding_gradient(dy, order, vocabulary, 3.0, out=base.clone(), accumulate=True)
    for extra, front in ((8, 0), (1, 0), (1, 1), (8, 3)):
        view = _beside(dy, extra, front)
        assert torch.equal(embedding.embedding_gradient(view, order, vocabulary, 3.0), want)
        assert torch.equal(embedding.embedding_gradient(view, order, vocabulary, 3.0, out=_beside(base, extra, front), accumulate=True), more)
