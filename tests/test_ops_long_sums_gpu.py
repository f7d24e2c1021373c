"""The gradients' sums over very many queries and rows: the tensor cores cut
off, and do not round, what falls below a sum's last bit, a loss that grows with
the number of steps where all terms have one sign. The logits here are 0 and the
number of rows a power of two, so that G is exact in 16 bits and the sums are all
that can be off.
"""
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def check(got, want, size):
    """size: the sum of the terms' magnitudes. A chunk of 64 K blocks (256 steps of
    16 terms) loses at most a last bit, 2^-23, a step; the chunks, shares and
    pieces are added up in FP32, 2^9 of them at most here; lse, G's FP32 steps and
    the factor take 2^-20; the result is rounded to half a step of its type."""
    import torch
    info = torch.finfo(got.dtype)
    bound = size * (256 * 2.0 ** -23 + 512 * U32 + 2.0 ** -20) + want.abs() * (info.eps / 2) * 1.01 + 1e-7
    off = float(((got.double() - want).abs() / bound).max())
    assert off <= 1.0, 'off by %.3g of the bound' % off


@pytest.mark.parametrize('dtype', ['float16', 'bfloat16'])
def test_rows_gradient_over_two_million_queries(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    nq, rows, dims, scale = (1 << 21) + 77, 4, 8, 2.0 ** -8
    g = torch.Generator(device='cuda')
    g.manual_seed(1)
    x = (0.5 + 0.5 * torch.rand((nq, dims), generator=g, device='cuda')).to(getattr(torch, dtype))
    w = torch.zeros((rows, dims), device='cuda', dtype=x.dtype)
    t = torch.zeros((nq,), dtype=torch.int64, device='cuda')
    _, lse = pb.softmax_loss(x, w, t, scale=scale)
    _, dw = pb.softmax_loss_grad(x, w, t, lse, scale=scale, need_queries=False)
    total = scale * x.double().sum(dim=0)
    part = torch.tensor([-0.75, 0.25, 0.25, 0.25], dtype=torch.float64, device='cuda')
    want = part[:, None] * total
    check(dw, want, want.abs())


@pytest.mark.parametrize('dtype', ['float16', 'bfloat16'])
def test_queries_gradient_over_a_million_rows(cuda, dtype):
    # 17 tiles of 256 queries x 256 dimensions: four shares of 262,144 rows each
    import torch
    import pgvector_b200 as pb
    nq, rows, dims = 256, 1 << 20, 4352
    g = torch.Generator(device='cuda')
    g.manual_seed(2)
    w = torch.empty((rows, dims), device='cuda', dtype=getattr(torch, dtype))
    total = torch.zeros((dims,), dtype=torch.float64, device='cuda')
    for i in range(0, rows, 1 << 16):
        w[i:i + (1 << 16)] = 0.5 + 0.5 * torch.rand((1 << 16, dims), generator=g, device='cuda')
        total += w[i:i + (1 << 16)].double().sum(dim=0)
    x = torch.zeros((nq, dims), device='cuda', dtype=w.dtype)
    t = torch.randint(0, rows, (nq,), generator=g, device='cuda')
    _, lse = pb.softmax_loss(x, w, t)
    dx, _ = pb.softmax_loss_grad(x, w, t, lse, need_rows=False)
    mean = total / rows
    check(dx, mean - w[t].double(), (mean + w[t].double()))
