"""The operators over a shard's rows against their formulas in 64 bits: softmax
loss and gradients, the quantizer to E4M3 with a scale per block of 128, and
products in that form. Tolerances are error bounds: every sum of n terms in
FP32 is off by at most n roundings of the sum of the terms' magnitudes, every
rounding to a type by half its step (finfo.eps / 2) or, below its normal
range, half its smallest step.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = ['f32', 'f16', 'bf16']


def torch_type(name):
    import torch
    return {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}[name]


def half_step(dtype, value):
    """Half a step of `dtype` at |value| (64-bit tensor)."""
    import torch
    info = torch.finfo(dtype)
    return value.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def within(got, want, bound):
    diff = (got.double() - want).abs()
    worst = (diff / bound).max().item() if diff.numel() else 0.0
    assert bool((diff <= bound).all()), 'off by %.3g of the bound' % worst


# ---------------------------------------------------------------- softmax loss

def loss_inputs(nq, rows, dims, dtype, seed, unit=True, none=0.1):
    import torch
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    w = torch.randn((rows, dims), generator=g, device='cuda')
    t = torch.randint(0, rows, (nq,), generator=g, device='cuda')
    x = w[t] + torch.randn((nq, dims), generator=g, device='cuda')
    if unit:
        w /= w.norm(dim=1, keepdim=True).clamp_min(1e-6)
        x /= x.norm(dim=1, keepdim=True).clamp_min(1e-6)
    t[torch.rand((nq,), generator=g, device='cuda') < none] = -1
    grad = torch.rand((nq,), generator=g, device='cuda') + 0.25
    return x.to(torch_type(dtype)), w.to(torch_type(dtype)), t, grad


def loss_reference(x, w, t, grad, scale):
    """Values and error bounds in 64 bits."""
    import torch
    dtype = x.dtype
    nq, rows, dims = x.shape[0], w.shape[0], x.shape[1]
    kept = (t >= 0) & (t < rows)
    xd = torch.where(kept[:, None], x.double(), torch.zeros((), dtype=torch.float64, device='cuda'))
    xa, wd = x.double(), w.double()
    logit = xa @ wd.t() * scale
    lse = torch.logsumexp(logit, dim=1)
    at = t.clamp(0, rows - 1)
    loss = torch.where(kept, lse - logit.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    # a logit: dims products (FP32 operands: as two 11-bit terms each, three
    # products of four) and sums, the scale, conversion to base 2
    e = (abs(scale) * (xa.abs() @ wd.abs().t())).amax(dim=1) * ((dims + 16) * 2.0 ** -23) + 2.0 ** -22
    # the sum of exponentials: positive terms, each within 2^-21 of its value (ex2.approx: 2^-22)
    lse_bound = e + 2.0 ** -20 + (math.log2(rows + 1) + 2 + lse.abs()) * 2.0 ** -22
    loss_bound = torch.where(kept, 2 * e + 2.0 ** -20 + (math.log2(rows + 1) + 4 + 2 * lse.abs()) * 2.0 ** -22,
                             torch.zeros_like(e))
    p = torch.exp(logit - lse[:, None])
    hot = torch.zeros_like(p)
    hot[torch.arange(nq, device='cuda'), at] = 1.0
    gk = torch.where(kept, grad.double(), torch.zeros_like(lse))
    G = gk[:, None] * (p - hot)
    # exp(l - lse): the logit's and lse's errors; then G is held in 16 bits,
    # or in two FP16 terms (22 bits); FP16 terms are scaled so that the
    # largest |grad| is 2^14 at least, steps of 2^-24 below their range
    u = 2.0 ** -21 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    top = grad.abs().max().double()
    dG = gk.abs()[:, None] * p * (2 * e + 2.0 ** -19 + lse.abs() * 2.0 ** -22)[:, None] + G.abs() * u \
        + (top * 2.0 ** -38 if dtype != torch.bfloat16 else 0.0)
    dG = torch.where(kept[:, None], dG, torch.zeros_like(dG))
    dx, dw = scale * (G @ wd), scale * (G.t() @ xd)
    more = 2.0 ** -20 if dtype == torch.float32 else 0.0
    dx_bound = abs(scale) * (dG @ wd.abs() + (G.abs() @ wd.abs()) * ((rows + 16) * U32 + more)) + half_step(dtype, dx)
    dw_bound = abs(scale) * (dG.t() @ xd.abs() + (G.abs().t() @ xd.abs()) * ((nq + 16) * U32 + more)) + half_step(dtype, dw)
    return dict(loss=(loss, loss_bound), lse=(lse, lse_bound), dx=(dx, dx_bound * 1.01), dw=(dw, dw_bound * 1.01))


def check_loss(x, w, t, grad, scale):
    import pgvector_b200 as pb
    ref = loss_reference(x, w, t, grad, scale)
    loss, lse = pb.softmax_loss(x, w, t, scale=scale)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=scale)
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and dx.is_contiguous() and dw.is_contiguous()
    for name, got in (('lse', lse), ('loss', loss), ('dx', dx), ('dw', dw)):
        within(got, *ref[name])
    return loss, lse, dx, dw


SIZES = [(1, 1, 1), (1, 2, 3), (2, 7, 8), (3, 64, 16), (5, 255, 40), (1, 256, 64), (33, 257, 129), (64, 1000, 200),
         (128, 512, 128), (129, 513, 65), (255, 300, 96), (257, 3000, 33), (300, 70001, 24), (1, 50000, 768),
         (17, 1025, 1000), (700, 130, 520)]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('nq,rows,dims', SIZES)
def test_loss_and_gradients(cuda, dtype, nq, rows, dims):
    x, w, t, g = loss_inputs(nq, rows, dims, dtype, seed=nq + rows + dims)
    check_loss(x, w, t, g, scale=12.5)


@pytest.mark.parametrize('dtype', TYPES)
def test_gradients_over_several_pieces_of_the_rows(cuda, dtype):
    # more than the 512 MB that a piece's part of the logits' gradient takes
    x, w, t, g = loss_inputs(2100, 140001, 16, dtype, seed=18)
    check_loss(x, w, t, g, scale=12.5)


def test_the_loss_of_a_batch_in_several_launches(cuda):
    # 1,300 queries against 3,000,001 rows: partial sums for 1,280 queries at a time
    import torch
    import pgvector_b200 as pb
    x, w, t, _ = loss_inputs(1300, 3000001, 16, 'bf16', seed=19)
    loss, lse = pb.softmax_loss(x, w, t, scale=9.0)
    for part in (slice(0, 700), slice(700, 1300)):
        a, b = pb.softmax_loss(x[part], w, t[part].contiguous(), scale=9.0)
        assert torch.equal(a, loss[part]) and torch.equal(b, lse[part])


@pytest.mark.parametrize('dtype', TYPES)
def test_loss_large_and_odd_scales(cuda, dtype):
    x, w, t, g = loss_inputs(40, 900, 72, dtype, seed=3)
    for scale in (0.0, -3.0, 100.0):
        check_loss(x, w, t, g, scale)
    x, w, t, g = loss_inputs(40, 900, 72, dtype, seed=4, unit=False)
    check_loss(x, w, t, g * 1e-3, 0.125)


@pytest.mark.parametrize('dtype', TYPES)
def test_loss_strided_and_misaligned_operands(cuda, dtype):
    import torch
    x, w, t, g = loss_inputs(50, 700, 72, dtype, seed=5)
    want = check_loss(x, w, t, g, 9.0)
    hx = torch.full((50, 101), float('nan'), dtype=x.dtype, device='cuda')
    hw = torch.full((700, 83), float('nan'), dtype=w.dtype, device='cuda')
    hx[:, 3:75], hw[:, 1:73] = x, w
    hw2 = torch.full((700, 128), float('nan'), dtype=w.dtype, device='cuda')
    hw2[:, 8:80] = w
    for a, b in ((hx[:, 3:75], w), (x, hw[:, 1:73]), (hx[:, 3:75], hw2[:, 8:80])):
        got = check_loss(a, b, t, g, 9.0)
        for p, q in zip(got, want):
            assert torch.equal(p, q)


@pytest.mark.parametrize('dtype', TYPES)
def test_queries_without_a_target_add_nothing(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    x, w, t, g = loss_inputs(70, 500, 48, dtype, seed=6, none=0.0)
    t[::3] = -1
    t[1] = -(1 << 62)
    bad = x.clone()
    bad[::3] = float('nan')
    bad[3] = float('inf')
    bad[6] = -torch.finfo(x.dtype).max
    bad[1] = float('nan')
    loss, lse = pb.softmax_loss(x, w, t, scale=5.0)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=5.0)
    none = t < 0
    loss2, lse2 = pb.softmax_loss(bad, w, t, scale=5.0)
    dx2, dw2 = pb.softmax_loss_grad(bad, w, t, lse2, grad=g, scale=5.0)
    assert bool((loss[none] == 0).all()) and bool((dx[none] == 0).all())
    assert torch.equal(loss, loss2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    assert torch.equal(lse[~none], lse2[~none]) and bool(torch.isnan(lse2[0]))
    # none at all
    t[:] = -1
    loss, lse = pb.softmax_loss(x, w, t, scale=5.0)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=5.0)
    assert not loss.any() and not dx.any() and not dw.any()
    within(lse, torch.logsumexp(x.double() @ w.double().t() * 5.0, dim=1), torch.full_like(lse, 1e-3).double())


@pytest.mark.parametrize('dtype', TYPES)
def test_a_target_past_the_rows(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    x, w, t, g = loss_inputs(9, 300, 32, dtype, seed=7, none=0.0)
    ok = check_loss(x, w, t, g, 4.0)
    t[2], t[5] = 300, 1 << 40
    status = torch.full((9,), 77, dtype=torch.int32, device='cuda')
    loss, lse = pb.softmax_loss(x, w, t, scale=4.0, status=status)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=4.0)
    bad = torch.zeros(9, dtype=torch.bool, device='cuda')
    bad[2] = bad[5] = True
    assert status.tolist() == [1 if b else 0 for b in bad.tolist()]
    assert bool(torch.isnan(loss[bad]).all()) and torch.equal(loss[~bad], ok[0][~bad])
    assert not dx[bad].any() and torch.equal(dx[~bad], ok[2][~bad])
    assert bool(torch.isfinite(dw).all())


@pytest.mark.parametrize('dtype', TYPES)
def test_non_finite_values_stay_with_what_holds_them(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    x, w, t, g = loss_inputs(40, 600, 64, dtype, seed=8, none=0.0)
    ok = check_loss(x, w, t, g, 4.0)
    x2 = x.clone()
    x2[7, 3] = float('nan')
    loss, lse = pb.softmax_loss(x2, w, t, scale=4.0)
    dx, dw = pb.softmax_loss_grad(x2, w, t, lse, grad=g, scale=4.0)
    other = torch.arange(40, device='cuda') != 7
    assert bool(torch.isnan(loss[7])) and bool(torch.isnan(lse[7])) and bool(torch.isnan(dx[7]).all())
    assert torch.equal(loss[other], ok[0][other]) and torch.equal(dx[other], ok[2][other])
    if dtype == 'f32':   # (held as two terms: an infinite value counts as a NaN)
        w2 = w.clone()
        w2[11, 5] = float('inf')
        loss, lse = pb.softmax_loss(x, w2, t, scale=4.0)
        assert bool(torch.isnan(lse).all())
        return
    # a row of -inf has probability 0 for queries of positive values: the others' loss stays
    xp, wp = x.abs() + 0.01, w.clone()
    wp[11] = float('-inf')
    t2 = torch.where(t == 11, 12, t)
    keep = torch.arange(600, device='cuda') != 11
    ref, _ = pb.softmax_loss(xp, wp[keep].contiguous(), torch.where(t2 > 11, t2 - 1, t2), scale=4.0)
    got, _ = pb.softmax_loss(xp, wp, t2, scale=4.0)
    within(got, ref.double(), torch.full_like(ref, 1e-4).double())


@pytest.mark.parametrize('dtype', TYPES)
def test_logits_far_apart(cuda, dtype):
    # one logit above the others by more than exp can hold, and below
    import torch
    import pgvector_b200 as pb
    x = torch.zeros((4, 16), device='cuda', dtype=torch_type(dtype))
    w = torch.zeros((600, 16), device='cuda', dtype=torch_type(dtype))
    x[:, 0] = torch.tensor([1.0, -1.0, 2.0, 0.0])
    w[300, 0], w[599, 0] = 500.0, -500.0
    t = torch.tensor([300, 599, 0, 599], device='cuda')
    loss, lse = pb.softmax_loss(x, w, t)
    want = torch.tensor([0.0, 0.0, 1000.0, math.log(600)], device='cuda')
    within(loss, want.double(), torch.full((4,), 1e-3, device='cuda').double())
    dx, dw = pb.softmax_loss_grad(x, w, t, lse)
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all())
    # p = exp(1000 - lse) with lse held in FP32: off by its half step and the logit's, in base 2 and e
    off = 1000 * 2.0 ** -22
    assert abs(float(dx[2, 0]) - 500.0) <= 500 * (off + torch.finfo(x.dtype).eps)
    assert abs(float(dw[300, 0]) - 2.0) <= 4 * (off + torch.finfo(x.dtype).eps)


@pytest.mark.parametrize('dtype', TYPES)
def test_weights_of_very_different_size(cuda, dtype):
    import torch
    x, w, t, g = loss_inputs(60, 400, 56, dtype, seed=9)
    g = torch.where(torch.arange(60, device='cuda') % 2 == 0, g, torch.zeros_like(g))
    g[4] = -2.0
    check_loss(x, w, t, g, 8.0)
    check_loss(x, w, t, g * 2.0 ** -12, 8.0)
    check_loss(x, w, t, torch.zeros_like(g), 8.0)


def test_fp32_operands_keep_their_bits(cuda):
    # values whose low bits FP16 and BF16 lose: the loss moves by them
    import torch
    x, w, t, g = loss_inputs(30, 500, 64, 'f32', seed=10, unit=False)
    check_loss(x * 1e-4, w * 1e3, t, g, 1.0)
    check_loss(x * 1e4, w * 1e-6, t, g, 10.0)


@pytest.mark.parametrize('dtype', TYPES)
def test_only_the_gradients_asked_for(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    x, w, t, g = loss_inputs(65, 800, 40, dtype, seed=11)
    _, lse = pb.softmax_loss(x, w, t, scale=6.0)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=6.0)
    a, none = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=6.0, need_rows=False)
    assert none is None and torch.equal(a, dx)
    none, b = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=6.0, need_queries=False)
    assert none is None and torch.equal(b, dw)
    ones, _ = pb.softmax_loss_grad(x, w, t, lse, scale=6.0)
    same, _ = pb.softmax_loss_grad(x, w, t, lse, grad=torch.ones_like(g), scale=6.0)
    assert torch.equal(ones, same)
    dx, dw = pb.softmax_loss_grad(x[:0], w, t[:0], lse[:0], scale=6.0)
    assert dx.shape == (0, 40) and not dw.any()


def test_gradients_against_differences(cuda):
    # along a direction v: (L(x + h v) - L(x - h v)) / 2h. Its truncation is
    # h^2/6 |L'''|, and a log-sum-exp's third derivative is at most
    # R^3 / (6 sqrt 3) for slopes within a range R.
    import torch
    import pgvector_b200 as pb
    nq, rows, dims, scale, h = 20, 400, 32, 3.0, 2.0 ** -5
    x, w, t, g = loss_inputs(nq, rows, dims, 'f32', seed=12)
    _, lse = pb.softmax_loss(x, w, t, scale=scale)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=scale)
    gen = torch.Generator(device='cuda')
    gen.manual_seed(13)
    for wrt in ('x', 'w'):
        v = torch.randn((x if wrt == 'x' else w).shape, generator=gen, device='cuda')
        v /= v.norm(dim=1, keepdim=True)
        up = pb.softmax_loss(x + h * v if wrt == 'x' else x, w + h * v if wrt == 'w' else w, t, scale=scale)[0]
        down = pb.softmax_loss(x - h * v if wrt == 'x' else x, w - h * v if wrt == 'w' else w, t, scale=scale)[0]
        diff = ((up.double() - down.double()) * g).sum() / (2 * h)
        slopes = scale * (v.double() @ w.double().t() if wrt == 'x' else x.double() @ v.double().t())
        r = slopes.amax(dim=1) - slopes.amin(dim=1)
        kept = (t >= 0).double()
        truncation = (h * h / 6 * r ** 3 / (6 * math.sqrt(3)) * g * kept).sum()
        bound = loss_reference(x, w, t, g, scale)['loss'][1] * 1.5   # |x|, |w| grow by h at most
        rounding = (bound * g).sum() / h + 1e-4
        want = ((dx if wrt == 'x' else dw).double() * v).sum()
        assert abs(float(diff - want)) <= float(truncation + rounding)
        assert abs(float(want)) > 10 * float(truncation + rounding)


@pytest.mark.parametrize('dtype', TYPES)
def test_loss_calls_repeat_and_run_side_by_side(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    a = loss_inputs(200, 5000, 72, dtype, seed=14)
    b = loss_inputs(90, 7000, 72, dtype, seed=15)
    torch.cuda.synchronize()

    def both(args, stream=None):
        x, w, t, g = args
        loss, lse = pb.softmax_loss(x, w, t, scale=7.0, stream=stream)
        return (loss, lse) + pb.softmax_loss_grad(x, w, t, lse, grad=g, scale=7.0, stream=stream)

    want = [both(a), both(b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        got.append([both(a, s1), both(b, s2)])
    torch.cuda.synchronize()
    for pair in got:
        for p, q in zip(pair, want):
            for u, v in zip(p, q):
                assert torch.equal(u, v)


@pytest.mark.parametrize('dtype', TYPES)
def test_loss_in_captured_graphs(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    x, w, t, g = loss_inputs(100, 3000, 64, dtype, seed=16)
    x2, w2, t2, g2 = loss_inputs(100, 3000, 64, dtype, seed=17)
    bufs = [v.clone() for v in (x, w, t, g)]

    def step():
        loss, lse = pb.softmax_loss(bufs[0], bufs[1], bufs[2], scale=7.0)
        return (loss, lse) + pb.softmax_loss_grad(bufs[0], bufs[1], bufs[2], lse, grad=bufs[3], scale=7.0)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for args in ((x, w, t, g), (x2, w2, t2, g2)):
        for buf, v in zip(bufs, args):
            buf.copy_(v)
        want = step()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for u, v in zip(out, want):
                assert torch.equal(u, v)


CAPTURE_FIRST = r"""
import sys
sys.path.insert(0, %r)
import torch
import pgvector_b200 as pb
x = torch.randn((100, 64), device='cuda')
w = torch.randn((900, 64), device='cuda')
t = torch.arange(100, device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    loss, lse = pb.softmax_loss(x, w, t)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse)
    a, sa = pb.quantize_blocks(x)
    b, sb = pb.quantize_blocks(w, square=True)
    out = [pb.matmul_blocks(a[:m], sa[:m], b, sb) for m in (1, 20, 100)]
graph.replay()
torch.cuda.synchronize()
want = pb.softmax_loss(x, w, t)
assert torch.equal(loss, want[0]) and torch.equal(lse, want[1])
for u, v in zip((dx, dw), pb.softmax_loss_grad(x, w, t, lse)):
    assert torch.equal(u, v)
for m, o in zip((1, 20, 100), out):
    assert torch.equal(o, pb.matmul_blocks(a[:m], sa[:m], b, sb))
print('captured')
"""


def test_first_calls_of_a_process_can_be_captured(cuda):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, '-c', CAPTURE_FIRST % root], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and 'captured' in out.stdout, out.stderr


# ---------------------------------------------------------------- blocks of E4M3

def e4m3_values():
    c = np.arange(127)
    return np.where(c < 8, c * 2.0 ** -9, (8 + (c & 7)) * 2.0 ** ((c >> 3) - 10.0))


def quantize_reference(x, square):
    """(codes uint8, scales float32) of a float32 array, step by step as annb200.h says."""
    m, k = x.shape
    kb, h = (k + 127) // 128, 128 if square else 1
    mb = (m + h - 1) // h
    pad = np.zeros((mb * h, kb * 128), np.float32)
    pad[:m, :k] = x
    v = pad.reshape(mb, h, kb, 128)
    a = np.abs(v).max(axis=(1, 3))
    a = np.where(a == 0, np.float32(448), np.maximum(a, np.float32(2.0 ** -100))).astype(np.float32)
    inverse = np.float32(448) / a
    u = np.abs(v * inverse[:, None, :, None]).astype(np.float32).astype(np.float64)
    table = e4m3_values()
    i = np.clip(np.searchsorted(table, u), 1, 126)
    below, above = table[i - 1], table[i]
    up = (u - below > above - u) | ((u - below == above - u) & (i % 2 == 0))
    code = (np.where(up, i, i - 1) + 128 * np.signbit(v)).astype(np.uint8)
    return code.reshape(mb * h, -1)[:m, :k], a / np.float32(448)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('square', [False, True])
@pytest.mark.parametrize('m,k', [(1, 1), (1, 127), (3, 128), (5, 129), (127, 15), (128, 256), (129, 384), (300, 1000),
                                 (1, 4097), (1000, 40), (257, 768)])
def test_quantize_bits(cuda, dtype, square, m, k):
    import torch
    import pgvector_b200 as pb
    rng = np.random.default_rng(m * 5 + k)
    x = rng.standard_normal((m, k)).astype(np.float32) * np.exp2(rng.integers(-6, 6, (m, 1))).astype(np.float32)
    x[rng.random((m, k)) < 0.1] = 0.0
    x[m // 2, : min(k, 128)] = 0.0
    # ties: absmax 448 makes the scale 1, odd multiples of half a step follow
    if k >= 8:
        x[0, : min(k, 128)] = 0.0
        x[0, :8] = [448.0, 17.0, 19.0, -21.0, 2.0 ** -10, 3 * 2.0 ** -10, -2.0 ** -11, 0.0625 * 1.0625]
    xt = torch.from_numpy(x).to(torch_type(dtype)).cuda()
    codes, scales = pb.quantize_blocks(xt, square=square)
    want, ws = quantize_reference(xt.float().cpu().numpy(), square)
    assert codes.shape == (m, k) and codes.stride(0) % 16 == 0
    assert np.array_equal(scales.cpu().numpy(), ws)
    assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), want)


@pytest.mark.parametrize('dtype', TYPES)
def test_quantize_strides_padding_and_extremes(cuda, dtype):
    import torch
    import pgvector_b200 as pb
    from pgvector_b200._lib import load
    dt = torch_type(dtype)
    gen = torch.Generator(device='cuda')
    gen.manual_seed(20)
    held = torch.randn((70, 333), generator=gen, device='cuda').to(dt)
    x = held[:, 7:307]
    for square in (False, True):
        codes, scales = pb.quantize_blocks(x, square=square)
        c2, s2 = pb.quantize_blocks(x.contiguous(), square=square)
        assert torch.equal(codes.view(torch.uint8), c2.view(torch.uint8)) and torch.equal(scales, s2)
    # the bytes up to a multiple of 16 are zeroed, the rest of a longer code row is left as it was
    out = torch.full((70, 320 + 32), 0xaa, dtype=torch.uint8, device='cuda')
    sc = torch.empty((70, 3), dtype=torch.float32, device='cuda')
    types = {'f32': pb.F32, 'f16': pb.F16, 'bf16': pb.BF16}
    st = torch.cuda.current_stream().cuda_stream
    assert load().AnnB200QuantizeBlocks(types[dtype], x.data_ptr(), 333, 70, 300, 0, out.data_ptr(), 352,
                                        sc.data_ptr(), st) == 0
    codes, _ = pb.quantize_blocks(x)
    torch.cuda.synchronize()
    assert torch.equal(out[:, :300], codes.view(torch.uint8))
    assert bool((out[:, 300:304] == 0).all()) and bool((out[:, 304:] == 0xaa).all())
    # tiny and huge blocks
    info = torch.finfo(dt)
    e = torch.zeros((4, 256), dtype=dt, device='cuda')
    e[0, :128] = info.tiny
    e[1, 5] = info.smallest_normal * info.eps     # the smallest value there is
    e[2] = info.max
    e[3, 200] = -info.max
    codes, scales = pb.quantize_blocks(e)
    want, ws = quantize_reference(e.float().cpu().numpy(), False)
    assert np.array_equal(scales.cpu().numpy(), ws)
    assert np.array_equal(codes.view(torch.uint8).cpu().numpy() & 0x7f, want & 0x7f)


@pytest.mark.parametrize('square', [False, True])
def test_quantize_non_finite(cuda, square):
    import torch
    import pgvector_b200 as pb
    x = torch.ones((130, 300), device='cuda')
    x[1, 130] = float('nan')
    x[129, 299] = float('-inf')
    codes, scales = pb.quantize_blocks(x, square=square)
    v = codes.float()
    nan_rows = slice(0, 128) if square else slice(1, 2)
    inf_rows = slice(128, 130) if square else slice(129, 130)
    assert bool(torch.isnan(v[nan_rows, 128:256]).all())
    assert bool(torch.isnan(scales[0 if square else 1, 1])) and bool(torch.isinf(scales[1 if square else 129, 2]))
    assert bool(torch.isnan(v[129, 299])) and bool((v[inf_rows, 256:299] == 0).all())
    rest = torch.ones((130, 300), dtype=torch.bool, device='cuda')
    rest[nan_rows, 128:256] = False
    rest[inf_rows, 256:] = False
    assert bool((v[rest] == 448).all())


def operand(m, k, seed, square):
    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    x = torch.randn((m, k), generator=g, device='cuda') * torch.exp2(
        torch.randint(-4, 5, (1, k), generator=g, device='cuda').float())
    return pb.quantize_blocks(x, square=square)


def decoded(codes, scales):
    m, k = codes.shape
    s = scales.double().repeat_interleave(128, 1)[:, :k]
    if scales.shape[0] != m:
        s = s.repeat_interleave(128, 0)[:m]
    return codes.double() * s


def check_matmul(a, sa, b, sb, out):
    import torch
    import pgvector_b200 as pb
    got = pb.matmul_blocks(a, sa, b, sb, dtype=torch_type(out))
    assert got.dtype == torch_type(out) and got.shape == (a.shape[0], b.shape[0])
    da, db = decoded(a, sa), decoded(b, sb)
    want = da @ db.t()
    # a block's sum of 128 products, the scales' product, their product, the sum over blocks
    k = a.shape[1]
    bound = (da.abs() @ db.abs().t()) * ((min(k, 128) + (k + 127) // 128 + 8) * 2.0 ** -23)
    within(got, want, (bound + half_step(torch_type(out), want)) * 1.01 + 1e-300)
    return got


MATMUL_SIZES = [(1, 1, 1), (1, 1, 127), (1, 300, 128), (1, 4096, 1024), (2, 129, 129), (3, 1000, 16), (4, 513, 700),
                (5, 255, 257), (8, 2000, 384), (16, 640, 1000), (17, 77, 2048), (33, 4097, 768), (64, 128, 128),
                (100, 1, 300), (127, 130, 500), (128, 256, 256), (129, 257, 130), (256, 256, 512), (300, 1, 64),
                (300, 1000, 1100), (513, 769, 640), (1030, 520, 96)]


@pytest.mark.parametrize('out', TYPES)
@pytest.mark.parametrize('m,n,k', MATMUL_SIZES)
def test_matmul(cuda, out, m, n, k):
    a, sa = operand(m, k, m + n, False)
    b, sb = operand(n, k, n + k, (m + n + k) % 2 == 0)
    check_matmul(a, sa, b, sb, out)


@pytest.mark.parametrize('m', [1, 3, 40, 300])
@pytest.mark.parametrize('square_a', [False, True])
@pytest.mark.parametrize('square_b', [False, True])
def test_matmul_scale_layouts(cuda, m, square_a, square_b):
    a, sa = operand(m, 400, 31, square_a)
    b, sb = operand(333, 400, 32, square_b)
    check_matmul(a, sa, b, sb, 'f32')


@pytest.mark.parametrize('m', [1, 6, 50, 290])
def test_matmul_ignores_bytes_past_k(cuda, m):
    import torch
    import pgvector_b200 as pb
    a, sa = operand(m, 200, 33, False)
    b, sb = operand(310, 200, 34, True)
    want = check_matmul(a, sa, b, sb, 'f32')
    ha = torch.full((m, 240), 0x7f, dtype=torch.uint8, device='cuda')   # E4M3's NaN
    hb = torch.full((310, 208), 0xff, dtype=torch.uint8, device='cuda')
    ha[:, 16:216], hb[:, :200] = a.view(torch.uint8), b.view(torch.uint8)
    got = pb.matmul_blocks(ha[:, 16:216], sa, hb[:, :200], sb)
    assert torch.equal(got, want)


@pytest.mark.parametrize('m', [1, 20, 300])
def test_matmul_non_finite(cuda, m):
    import torch
    import pgvector_b200 as pb
    a, sa = operand(m, 300, 35, False)
    b, sb = operand(200, 300, 36, False)
    want = check_matmul(a, sa, b, sb, 'f32')
    b = b.view(torch.uint8).clone()
    bb = torch.zeros((200, 304), dtype=torch.uint8, device='cuda')
    bb[:, :300] = b
    bb[17, 5] = 0x7f
    sb = sb.clone()
    sb[90, 1] = float('nan')
    got = pb.matmul_blocks(a, sa, bb[:, :300], sb)
    other = torch.ones(200, dtype=torch.bool, device='cuda')
    other[17] = other[90] = False
    assert bool(torch.isnan(got[:, ~other]).all()) and torch.equal(got[:, other], want[:, other])


def test_matmul_empty(cuda):
    import torch
    import pgvector_b200 as pb
    a, sa = operand(4, 64, 37, False)
    assert pb.matmul_blocks(a[:0], sa[:0], a, sa).shape == (0, 4)
    assert pb.matmul_blocks(a, sa, a[:0], sa[:0]).shape == (4, 0)
    e, se = a[:, :0], sa[:, :0].contiguous()
    assert not pb.matmul_blocks(e, se, e, se).any()


def test_matmul_past_32_bit_offsets(cuda):
    # 4.3 GB of output: elements past 2^31 and bytes past 2^32
    import torch
    import pgvector_b200 as pb
    a, sa = operand(70, 64, 38, False)
    b, sb = operand(32000000, 64, 39, False)
    got = pb.matmul_blocks(a, sa, b, sb, dtype=torch.float16)
    for at in (0, 12345678, 31999000):
        part = pb.matmul_blocks(a, sa, b[at:at + 1000], sb[at:at + 1000], dtype=torch.float16)
        want = decoded(a, sa) @ decoded(b[at:at + 1000], sb[at:at + 1000]).t()
        assert torch.equal(got[:, at:at + 1000], part)
        within(part, want, want.abs() * 2.0 ** -10 + 1e-3)


def test_blocks_repeat_and_run_side_by_side(cuda):
    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(40)
    x = torch.randn((260, 900), generator=g, device='cuda')
    w = torch.randn((3000, 900), generator=g, device='cuda')

    def both(stream=None):
        a, sa = pb.quantize_blocks(x, stream=stream)
        b, sb = pb.quantize_blocks(w, square=True, stream=stream)
        return [pb.matmul_blocks(a[:m], sa[:m], b, sb, stream=stream) for m in (1, 3, 60, 260)]

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [both(s) for _ in range(3) for s in streams]
    torch.cuda.synchronize()
    for outs in got:
        for u, v in zip(outs, want):
            assert torch.equal(u, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    x.copy_(torch.randn((260, 900), generator=g, device='cuda'))
    want = both()
    graph.replay()
    torch.cuda.synchronize()
    for u, v in zip(outs, want):
        assert torch.equal(u, v)


# ---------------------------------------------------------------- together

def test_rows_are_trained_then_served_in_blocks(cuda):
    """A shard's rows trained by the loss over all of them, stored as blocks of
    E4M3, and scored for one query and for a batch; the shard's own search
    finds the same best row."""
    import torch
    import pgvector_b200 as pb
    g = torch.Generator(device='cuda')
    g.manual_seed(50)
    rows, dims, nq, scale = 3000, 96, 64, 10.0
    w = torch.nn.functional.normalize(torch.randn((rows, dims), generator=g, device='cuda'), dim=1)
    proj = torch.randn((dims, dims), generator=g, device='cuda').mul_(dims ** -0.5).requires_grad_()
    feats = torch.randn((nq, dims), generator=g, device='cuda')
    t = torch.randint(0, rows, (nq,), generator=g, device='cuda')
    t[3] = -1
    for _ in range(3):
        x = feats @ proj
        loss, lse = pb.softmax_loss(x.detach(), w, t, scale=scale)
        weight = torch.full((nq,), 1.0 / nq, device='cuda')
        dx, dw = pb.softmax_loss_grad(x.detach(), w, t, lse, grad=weight, scale=scale)
        ref = loss_reference(x.detach(), w, t, weight, scale)
        for name, got in (('lse', lse), ('loss', loss), ('dx', dx), ('dw', dw)):
            within(got, *ref[name])
        proj.grad = None
        x.backward(dx)
        assert torch.isfinite(proj.grad).all()
        with torch.no_grad():
            proj -= 0.5 * proj.grad
            w -= 0.5 * dw
    q = (feats @ proj).detach().contiguous()
    codes, scales = pb.quantize_blocks(w)
    qc, qs = pb.quantize_blocks(q)
    batch = check_matmul(qc, qs, codes, scales, 'f32')
    for i in (0, 17):
        one = check_matmul(qc[i:i + 1], qs[i:i + 1], codes, scales, 'f32')
        within(one, batch[i:i + 1].double(), batch[i:i + 1].double().abs() * 2.0 ** -16 + 2.0 ** -10)
    # the search over the rows the codes stand for ranks them as the scores do
    held = decoded(codes, scales).float().contiguous()
    heldq = decoded(qc, qs).float().contiguous()
    shard = pb.Shard(pb.F32, dims, held)
    dist, ids, _ = shard.search(heldq, 1, pb.IP)
    torch.cuda.synchronize()
    best = batch.max(dim=1).values.double()
    within(-dist[:, 0], best, best.abs() * 2.0 ** -14 + 2.0 ** -8)
    shard.close()
