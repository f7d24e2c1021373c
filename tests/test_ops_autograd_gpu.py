"""The softmax loss as a part of an autograd graph."""
import pytest

pytestmark = pytest.mark.gpu


def inputs(dtype='float32', nq=50, rows=700, dims=40, seed=1):
    import torch
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    x = torch.randn((nq, dims), generator=g, device='cuda').to(getattr(torch, dtype)).requires_grad_()
    w = torch.randn((rows, dims), generator=g, device='cuda').to(getattr(torch, dtype)).requires_grad_()
    t = torch.randint(0, rows, (nq,), generator=g, device='cuda')
    t[4] = -1
    weight = torch.rand((nq,), generator=g, device='cuda') + 0.5
    return x, w, t, weight


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
def test_backward_is_the_gradient_call(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    x, w, t, weight = inputs(dtype)
    with torch.no_grad():
        loss0, lse0 = pb.softmax_loss(x, w, t, scale=0.3)
        assert not loss0.requires_grad
        dx, dw = pb.softmax_loss_grad(x, w, t, lse0, grad=weight, scale=0.3)
    loss, lse = pb.softmax_loss(x, w, t, scale=0.3)
    assert torch.equal(loss, loss0) and torch.equal(lse, lse0)
    (loss * weight).sum().backward()
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    # one weight for all, a gradient that is one number expanded; only one operand's gradient
    for need in (True, False):
        a, b = x.detach().requires_grad_(need), w.detach().requires_grad_(not need)
        pb.softmax_loss(a, b, t, scale=0.3)[0].mean().backward()
        ones = torch.full_like(weight, 1.0 / 50)
        dx, dw = pb.softmax_loss_grad(x, w, t, lse0, grad=ones, scale=0.3)
        assert torch.equal(a.grad, dx) if need else torch.equal(b.grad, dw)
        assert (b.grad if need else a.grad) is None


def test_it_adds_to_other_terms(cuda):
    import torch
    import pgvector_b200 as pb
    x, w, t, weight = inputs()
    proj = torch.eye(40, device='cuda').mul_(0.5).requires_grad_()
    y = x.detach() @ proj
    (pb.softmax_loss(y, w, t)[0].sum() + y.square().sum()).backward()
    with torch.no_grad():
        y = x @ proj
        dy, dw = pb.softmax_loss_grad(y, w, t, pb.softmax_loss(y, w, t)[1])
        want = x.double().t() @ (dy.double() + 2 * y.double())
        size = x.double().abs().t() @ (dy.double().abs() + 2 * y.double().abs())
    # two terms each rounded to FP32, then a sum over 50 queries, which torch may take in any order
    assert bool(((proj.grad.double() - want).abs() <= size * 60 * 2.0 ** -24 * 1.01).all())
    assert torch.equal(w.grad, dw)


def test_what_it_cannot_differentiate_is_refused(cuda):
    import torch
    import pgvector_b200 as pb
    x, w, t, _ = inputs()
    loss, lse = pb.softmax_loss(x, w, t)
    with pytest.raises(pb.AnnB200Error) as e:
        (loss.sum() + 1e-4 * lse.square().sum()).backward()
    assert e.value.status == pb.INVALID
    loss, lse = pb.softmax_loss(x, w, t)
    (loss.sum() + lse.detach().square().sum()).backward()
    loss, _ = pb.softmax_loss(x, w, t)
    first, = torch.autograd.grad(loss.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        first.sum().backward()
    # operands changed before the backward pass
    loss, _ = pb.softmax_loss(x, w, t)
    with torch.no_grad():
        w.mul_(0.5)
    with pytest.raises(RuntimeError):
        loss.sum().backward()


def test_on_another_stream_and_in_a_graph(cuda):
    import torch
    import pgvector_b200 as pb
    x, w, t, weight = inputs()
    with torch.no_grad():
        lse = pb.softmax_loss(x, w, t)[1]
        dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=weight)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    loss, _ = pb.softmax_loss(x, w, t, stream=side)
    side.synchronize()
    (loss * weight).sum().backward()
    torch.cuda.synchronize()
    assert torch.equal(x.grad, dx) and torch.equal(w.grad, dw)
    # a whole training step captured, no graph of the same leaves alive
    del loss
    x.grad = w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, _ = pb.softmax_loss(x, w, t)
        a, b = torch.autograd.grad((loss * weight).sum(), (x, w))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, dx) and torch.equal(b, dw)


def test_empty_batch(cuda):
    import torch
    import pgvector_b200 as pb
    x, w, t, _ = inputs()
    e = x.detach()[:0].requires_grad_()
    loss, _ = pb.softmax_loss(e, w, t[:0])
    loss.sum().backward()
    assert e.grad.shape == (0, 40) and not w.grad.any()
