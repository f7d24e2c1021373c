"""The softmax loss's gradients where the queries' weights differ by orders of
magnitude: each query's gradient is right relative to its own weight.

The rows hold nothing in the first half of the dimensions and the queries
nothing in the second, so every logit is 0, every probability 1 / rows, and

  dqueries_i = scale grad_i (mean of the rows - row_target)
  drows_j    = scale sum_i grad_i (1 / rows - [j = target(i)]) query_i

in closed form. The stored G of a query's other rows is one number, whose
rounding is not averaged out: losing FP32's second term shows, too.
"""
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
ROWS, DIMS, SCALE = 100003, 32, 5.0


def inputs(nq, dtype, seed):
    import torch
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    x = torch.zeros((nq, DIMS), device='cuda')
    w = torch.zeros((ROWS, DIMS), device='cuda')
    x[:, :DIMS // 2] = torch.randn((nq, DIMS // 2), generator=g, device='cuda')
    w[:, DIMS // 2:] = torch.randn((ROWS, DIMS // 2), generator=g, device='cuda')
    t = torch.randperm(ROWS, generator=g, device='cuda')[:nq]
    # from 1024 (a loss scale) down to 1e-7 of it, of any mantissa and sign
    grad = 1024.0 * torch.logspace(0, -7, nq, device='cuda') * (1.0 + torch.rand((nq,), generator=g, device='cuda'))
    grad[1::3] *= -1
    return x.to(dtype), w.to(dtype), t, grad


def half_step(dtype, value):
    import torch
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps / 2


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('nq', [24, 200])
def test_each_query_by_its_own_weight(cuda, dtype, nq):
    import math

    import torch
    import pgvector_b200 as pb
    dt = getattr(torch, dtype)
    x, w, t, grad = inputs(nq, dt, nq)
    none = nq - 3          # a query without a target, of a weight that must not count
    t[none], grad[none] = -1, 1e30
    loss, lse = pb.softmax_loss(x, w, t, scale=SCALE)
    kept = t >= 0
    g = torch.where(kept, grad.double(), torch.zeros((), dtype=torch.float64, device='cuda'))
    at = t.clamp_min(0)
    assert bool(((lse.double() - math.log(ROWS)).abs() <= 2.0 ** -20).all())
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=SCALE)
    xd, wd = x.double(), w.double()
    p = 1.0 / ROWS
    # G's entries: lse's half step (2^-21 at 11.5) and the FP32 steps from it to G (2^-21), then their rounding: one
    # step of a type, or of two FP16 terms (2^-21), at least 2^-39 of the weight with FP16 terms
    u = {'float32': 2.0 ** -21, 'float16': 2.0 ** -11, 'bfloat16': 2.0 ** -8}[dtype] + 2.0 ** -20
    floor = 0.0 if dtype == 'bfloat16' else 2.0 ** -39 * ROWS
    # the sums: chunks of up to 24 steps cut off at 2^-23 each and added in FP32; a share of the rows is 1,500 to
    # 3,200 of them, 25 chunks of 128 rows, 74 shares (one chunk of 200 steps for the 16-bit types)
    steps = 24 * 2.0 ** -23 + (25 + 74 + 8) * U32 if dtype == 'float32' else 200 * 2.0 ** -23 + (74 + 8) * U32
    want = SCALE * g[:, None] * (wd.mean(dim=0) - wd[at])
    spread = torch.stack([(wd - wd[i]).abs().mean(dim=0) for i in at])
    bound = SCALE * g.abs()[:, None] * (spread * (u + floor) + (wd.abs().mean(dim=0) + wd[at].abs()) * steps)
    bound = bound * 1.01 + half_step(dt, want)
    off = ((dx.double() - want).abs() / bound.clamp_min(1e-300))[kept]
    assert float(off.max()) <= 1.0, 'query %d off by %.3g of its bound' % (int(off.amax(dim=1).argmax()), float(off.max()))
    assert not dx[none].any()
    # the rows: every row, then those that are a target
    G = torch.full((ROWS, nq), p, dtype=torch.float64, device='cuda') * g
    G[at[kept], torch.nonzero(kept)[:, 0]] -= g[kept]
    want = SCALE * (G @ xd)
    top = float(g.abs().max()) * float(xd.abs().max())
    held = 0.0 if dtype == 'bfloat16' else 2.0 ** -38 * top
    small = torch.full_like(G, p)
    small[at[kept], torch.nonzero(kept)[:, 0]] = 1.0
    bound = SCALE * ((G.abs() @ xd.abs()) * (u + (nq + 16) * 2.0 ** -23)
                     + (floor / ROWS) * (g.abs() @ xd.abs())[None, :] + held * (small @ kept.double())[:, None])
    if dtype == 'float32':   # x times its weight as two FP16 terms
        bound += SCALE * (G.abs() @ xd.abs()) * 2.0 ** -21
    bound = bound * 1.01 + half_step(dt, want)
    off = (dw.double() - want).abs() / bound
    assert float(off.max()) <= 1.0, 'row %d off by %.3g of its bound' % (int(off.amax(dim=1).argmax()), float(off.max()))


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
def test_weights_times_a_power_of_two(cuda, dtype):
    # the same bits, moved: one query's gradient does not depend on the others' weights
    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(7)
    dt = getattr(torch, dtype)
    x = torch.randn((40, 48), generator=g, device='cuda').to(dt)
    w = torch.randn((3000, 48), generator=g, device='cuda').to(dt)
    t = torch.randint(0, 3000, (40,), generator=g, device='cuda')
    grad = torch.rand((40,), generator=g, device='cuda') + 0.5
    _, lse = pb.softmax_loss(x, w, t, scale=0.25)
    one, rows = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=0.25)
    power = torch.ones((40,), device='cuda')
    power[::2] = 1024.0
    two, _ = pb.softmax_loss_grad(x, w, t, lse, grad=grad * power, scale=0.25)
    assert torch.equal(two[1::2], one[1::2])
    normal = one.abs() >= torch.finfo(dt).tiny * 1024
    assert torch.equal((two.double() / power[:, None])[normal], one.double()[normal])
    # no weights at all are weights of one
    a = pb.softmax_loss_grad(x, w, t, lse, scale=0.25)
    b = pb.softmax_loss_grad(x, w, t, lse, grad=torch.ones_like(grad), scale=0.25)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # dqueries alone, drows alone
    a, _ = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=0.25, need_rows=False)
    _, b = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=0.25, need_queries=False)
    assert torch.equal(a, one) and torch.equal(b, rows)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_rows_near_the_largest_values(cuda, dtype):
    # rows of 2^120: their gradients are in range, and so is what leads to them
    import torch
    from test_ops_gpu import check_loss, loss_inputs
    x, w, t, g = loss_inputs(40, 900, 64, dtype, seed=11)
    _, _, dx, dw = check_loss(x * 2.0 ** -110, w * 2.0 ** 120, t, g, scale=2.0 ** -8)
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all()) and bool(dx.abs().max() > 2.0 ** 105)
