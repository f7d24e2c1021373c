"""The bounded waits of the operators' pair products: those that run out end
their kernel with NaN outputs, and the next call is right again.

ANN_B200_PIPELINE_WAIT_NS (read at every launch) shortens the waits; below one
try's sleep it also withholds the loads that they wait for. The drains after a
role has given up keep their 4 s limit, so each kernel here takes that long.
Nothing faults or hangs the GPU: every role leaves its loop.
"""
import pytest

pytestmark = pytest.mark.gpu


def operands(m, n, k, square):
    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(m + n + k)
    a = pb.quantize_blocks(torch.randn((m, k), generator=g, device='cuda'))
    b = pb.quantize_blocks(torch.randn((n, k), generator=g, device='cuda'), square=square)
    return a + b


# more K blocks than the stages and the two buffers of scales hold, several tiles a cluster
@pytest.mark.parametrize('m,square', [(20, False), (100, True), (300, False), (300, True)])
def test_product_whose_waits_run_out(cuda, monkeypatch, m, square):
    import torch
    import pgvector_b200 as pb
    args = operands(m, 30000, 2500, square)
    want = pb.matmul_blocks(*args)
    torch.cuda.synchronize()
    monkeypatch.setenv('ANN_B200_PIPELINE_WAIT_NS', '1')
    got = pb.matmul_blocks(*args)
    torch.cuda.synchronize()
    assert bool(torch.isnan(got).all())
    monkeypatch.delenv('ANN_B200_PIPELINE_WAIT_NS')
    assert torch.equal(pb.matmul_blocks(*args), want)


@pytest.mark.parametrize('nq,dtype', [(70, 'float32'), (300, 'float16')])
def test_loss_whose_waits_run_out(cuda, monkeypatch, nq, dtype):
    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(nq)
    x = torch.randn((nq, 200), generator=g, device='cuda').to(getattr(torch, dtype))
    w = torch.randn((20000, 200), generator=g, device='cuda').to(getattr(torch, dtype))
    t = torch.arange(nq, device='cuda')
    t[5] = -1

    def both(lse=None):
        loss, own = pb.softmax_loss(x, w, t, scale=0.1)
        return (loss, own) + pb.softmax_loss_grad(x, w, t, own if lse is None else lse, scale=0.1)

    want = both()
    torch.cuda.synchronize()
    monkeypatch.setenv('ANN_B200_PIPELINE_WAIT_NS', '1')
    loss, lse, dx, dw = both(want[1])
    torch.cuda.synchronize()
    assert bool(torch.isnan(lse).all())
    kept = t >= 0
    assert bool(torch.isnan(loss[kept]).all()) and bool(torch.isnan(dx[kept]).all()) and bool(torch.isnan(dw).all())
    assert not loss[~kept].any() and not dx[~kept].any()   # without a target: zero, whatever is known of it
    monkeypatch.delenv('ANN_B200_PIPELINE_WAIT_NS')
    for u, v in zip(both(), want):
        assert torch.equal(u, v)
