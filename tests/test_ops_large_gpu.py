"""The operators past 2^31 values of an operand or a result, with more than 1,000
dimensions, and called from several threads at once."""
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.mark.parametrize('n', [8000000, 7999999])   # results on 16-byte rows, and not
def test_wide_product_past_32_bit_offsets(cuda, n):
    import torch
    import pgvector_b200 as pb
    from test_ops_gpu import decoded, operand
    a, sa = operand(300, 16, 1, False)
    b, sb = operand(n, 16, 2, False)
    got = pb.matmul_blocks(a, sa, b, sb, dtype=torch.float16)
    assert got.numel() > 1 << 31
    for at in (0, 3333333, n - 1000):
        part = pb.matmul_blocks(a, sa, b[at:at + 1000], sb[at:at + 1000], dtype=torch.float16)
        assert torch.equal(got[:, at:at + 1000], part)
        want = decoded(a, sa) @ decoded(b[at:at + 1000], sb[at:at + 1000]).t()
        size = decoded(a, sa).abs() @ decoded(b[at:at + 1000], sb[at:at + 1000]).abs().t()
        bound = size * 32 * 2.0 ** -23 + want.abs() * 2.0 ** -11 * 1.01 + 2.0 ** -25
        assert bool(((part.double() - want).abs() <= bound).all())


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_gradients_past_32_bit_offsets(cuda, dtype):
    # rows and their gradient of 2.2e9 values each, off 16-byte boundaries, laid out in the workspace first
    import torch
    import pgvector_b200 as pb
    nq, rows, dims, scale = 4, 2200001, 1001, 6.0
    dt = getattr(torch, dtype)
    g = torch.Generator(device='cuda')
    g.manual_seed(3)
    w = torch.empty((rows, dims), dtype=dt, device='cuda')
    step = 100000
    for i in range(0, rows, step):
        part = torch.randn((min(step, rows - i), dims), generator=g, device='cuda')
        w[i:i + step] = part / part.norm(dim=1, keepdim=True)
    t = torch.tensor([0, rows - 1, -1, rows - 77], device='cuda')
    x = w[t.clamp_min(0)].clone()
    grad = torch.tensor([1.0, -0.5, 3.0, 2.0], device='cuda')
    loss, lse = pb.softmax_loss(x, w, t, scale=scale)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=scale)
    assert w.numel() > 1 << 31
    xd, kept = x.double(), t >= 0
    gk = torch.where(kept, grad, torch.zeros_like(grad)).double()[:, None]
    # errors of a logit, of G and of dX's sums: as in the small tests, the sums in chunks of 24 (FP32) or 256 steps of
    # the tensor cores, up to 455 chunks, 18 shares and 3 pieces
    e = scale * 1.01 * (dims + 16) * 2.0 ** -23 + 2.0 ** -22
    u = 2.0 ** -21 if dtype == 'float32' else 2.0 ** -11
    sums = (24 if dtype == 'float32' else 256) * 2.0 ** -23 + (455 + 18 + 3 + 8) * U32 + 2.0 ** -21
    total = torch.zeros((nq,), dtype=torch.float64, device='cuda')
    want, bound = torch.zeros_like(xd), torch.zeros_like(xd)
    for i in range(0, rows, step):
        wd = w[i:i + step].double()
        logit = scale * xd @ wd.t()
        total += torch.exp(logit).sum(dim=1)
        p = torch.exp(logit - lse.double()[:, None])
        hot = torch.zeros_like(p)
        for q in range(nq):
            if kept[q] and i <= int(t[q]) < i + wd.shape[0]:
                hot[q, int(t[q]) - i] = 1.0
        G = gk * (p - hot)
        dG = gk.abs() * p * (2 * e + 2.0 ** -19 + lse.double()[:, None].abs() * 2.0 ** -22) + G.abs() * u + gk.abs() * 2.0 ** -38
        want += scale * G @ wd
        bound += scale * (dG @ wd.abs() + sums * (G.abs() @ wd.abs()))
        drows = scale * G.t() @ xd
        off = scale * (dG.t() @ xd.abs() + G.abs().t() @ xd.abs() * 2.0 ** -20) + 2.0 ** -38 * scale * 2
        off = off * 1.01 + drows.abs() * torch.finfo(dt).eps / 2 + torch.finfo(dt).tiny * torch.finfo(dt).eps
        assert bool(((dw[i:i + step].double() - drows).abs() <= off).all()), 'rows from %d on' % i
    assert bool(((lse.double() - total.log()).abs() <= e + 2.0 ** -18).all())
    bound = bound * 1.01 + want.abs() * torch.finfo(dt).eps / 2 + torch.finfo(dt).tiny * torch.finfo(dt).eps
    assert bool(((dx.double() - want).abs() <= bound).all())
    assert not dx[2].any()


@pytest.mark.parametrize('dtype', ['f32', 'f16', 'bf16'])
@pytest.mark.parametrize('nq,rows,dims', [(30, 700, 1537), (65, 300, 4096), (300, 259, 1100), (3, 130, 65536)])
def test_many_dimensions(cuda, dtype, nq, rows, dims):
    from test_ops_gpu import check_loss, loss_inputs
    x, w, t, g = loss_inputs(nq, rows, dims, dtype, seed=dims)
    check_loss(x, w, t, g, scale=12.5)


def test_calls_from_several_threads(cuda):
    import threading

    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(5)
    jobs = []
    for i in range(4):
        x = torch.randn((90 + 40 * i, 64), generator=g, device='cuda')
        w = torch.randn((1000 + i, 64), generator=g, device='cuda')
        t = torch.randint(0, 1000, (x.shape[0],), generator=g, device='cuda')
        jobs.append((x, w, t))

    def run(job):
        x, w, t = job
        loss, lse = pb.softmax_loss(x, w, t, scale=0.2)
        a, sa = pb.quantize_blocks(x)
        b, sb = pb.quantize_blocks(w, square=True)
        return (loss, lse) + pb.softmax_loss_grad(x, w, t, lse, scale=0.2) + (pb.matmul_blocks(a, sa, b, sb),)

    want = [run(j) for j in jobs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = run(jobs[i])
                stream.synchronize()
                if not all(torch.equal(u, v) for u, v in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong
