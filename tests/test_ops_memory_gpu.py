"""The C calls keep to their memory: nothing is read of a workspace that the call
has not written, and nothing is written past a workspace or a result. Results
that may be left out are.
"""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

GUARD = 4096


class Room:
    """`size` bytes of 0xff (NaN in every type) between two guards."""

    def __init__(self, size):
        import torch
        self.held = torch.full((GUARD + size + GUARD,), 0xff, dtype=torch.uint8, device='cuda')
        self.size = size
        self.ptr = self.held.data_ptr() + GUARD
        assert self.ptr % 256 == 0

    def view(self, dtype, shape):
        return self.held[GUARD:GUARD + self.size].view(dtype).view(shape)

    def guards_are_whole(self):
        return bool((self.held[:GUARD] == 0xff).all()) and bool((self.held[GUARD + self.size:] == 0xff).all())


# aligned rows and not, one tile and several, several shares and pieces, up to 128 queries and more
SIZES = [(1, 1, 1), (1, 1000, 128), (3, 70, 9), (100, 900, 64), (128, 513, 201), (129, 700, 72), (300, 9000, 48),
         (70, 30000, 301), (2100, 140001, 8)]


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('nq,rows,dims', SIZES)
@pytest.mark.parametrize('weights', [False, True])
def test_loss_keeps_to_its_memory(cuda, dtype, nq, rows, dims, weights):
    import torch
    import pgvector_b200 as pb
    from pgvector_b200 import _abi
    from pgvector_b200._lib import load
    dt = getattr(torch, dtype)
    g = torch.Generator(device='cuda')
    g.manual_seed(nq + rows)
    x = (torch.randn((nq, dims), generator=g, device='cuda') * 0.3).to(dt)
    w = (torch.randn((rows, dims), generator=g, device='cuda') * 0.3).to(dt)
    t = torch.randint(0, rows, (nq,), generator=g, device='cuda')
    t[nq // 2] = -1 if nq > 1 else 0
    grad = torch.rand((nq,), generator=g, device='cuda') + 0.5 if weights else None
    loss, lse = pb.softmax_loss(x, w, t, scale=2.0)
    dx, dw = pb.softmax_loss_grad(x, w, t, lse, grad=grad, scale=2.0)
    out = {'loss': Room(4 * nq), 'lse': Room(4 * nq), 'dqueries': Room(nq * dims * x.element_size()),
           'drows': Room(rows * dims * x.element_size())}

    def job(**over):
        j = _abi.AnnB200LossJob({'float32': pb.F32, 'float16': pb.F16, 'bfloat16': pb.BF16}[dtype], dims, nq, 2.0, rows,
                                x.data_ptr(), dims, w.data_ptr(), dims, t.data_ptr())
        if weights:
            j.grad = grad.data_ptr()
        for k, r in over.items():
            setattr(j, k, r.ptr)
        return j

    def call(fn, which, **over):
        j = job(**over)
        need = (ctypes.c_uint64(), ctypes.c_uint64())
        assert load().AnnB200SoftmaxLossWorkspace(ctypes.byref(j), *[ctypes.byref(n) for n in need]) == 0
        room = Room(need[which].value)
        j.workspace, j.workspace_bytes = room.ptr, room.size
        assert getattr(load(), fn)(ctypes.byref(j), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert room.guards_are_whole()

    call('AnnB200SoftmaxLoss', 0, loss=out['loss'], lse=out['lse'])
    call('AnnB200SoftmaxLossGrad', 1, lse=out['lse'], dqueries=out['dqueries'], drows=out['drows'])
    for name, want in (('loss', loss), ('lse', lse), ('dqueries', dx), ('drows', dw)):
        assert out[name].guards_are_whole()
        assert torch.equal(out[name].view(want.dtype, want.shape), want)
    # one result alone
    for fn, which, name, want in (('AnnB200SoftmaxLoss', 0, 'loss', loss), ('AnnB200SoftmaxLoss', 0, 'lse', lse),
                                  ('AnnB200SoftmaxLossGrad', 1, 'dqueries', dx),
                                  ('AnnB200SoftmaxLossGrad', 1, 'drows', dw)):
        alone = Room(out[name].size)
        over = {name: alone} if which == 0 else {'lse': out['lse'], name: alone}
        call(fn, which, **over)
        assert alone.guards_are_whole() and torch.equal(alone.view(want.dtype, want.shape), want)


@pytest.mark.parametrize('m,n,k', [(1, 1, 1), (3, 77, 200), (8, 5000, 384), (9, 300, 130), (40, 1000, 1000),
                                   (128, 257, 64), (129, 255, 300), (300, 1001, 260), (513, 512, 128)])
@pytest.mark.parametrize('out', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('square', [False, True])
def test_blocks_keep_to_their_memory(cuda, m, n, k, out, square):
    import torch
    import pgvector_b200 as pb
    from pgvector_b200._lib import load
    g = torch.Generator(device='cuda')
    g.manual_seed(m + n + k)
    dt = getattr(torch, out)
    st = torch.cuda.current_stream().cuda_stream
    pad, kb = (k + 15) // 16 * 16, (k + 127) // 128
    types = {'float32': pb.F32, 'float16': pb.F16, 'bfloat16': pb.BF16}
    sides = []
    for rows, sq in ((m, False), (n, square)):
        x = torch.randn((rows, k), generator=g, device='cuda').to(dt)
        codes, scales = Room(rows * pad), Room(4 * kb * ((rows + 127) // 128 if sq else rows))
        assert load().AnnB200QuantizeBlocks(types[out], x.data_ptr(), k, rows, k, int(sq), codes.ptr, pad, scales.ptr,
                                            st) == 0
        torch.cuda.synchronize()
        assert codes.guards_are_whole() and scales.guards_are_whole()
        c, s = pb.quantize_blocks(x, square=sq)
        assert torch.equal(codes.view(torch.uint8, (rows, pad))[:, :k], c.view(torch.uint8))
        assert torch.equal(scales.view(torch.float32, s.shape), s)
        sides += [codes, scales, c, s]
    a, sa, ac, as_, b, sb, bc, bs = sides
    want = pb.matmul_blocks(ac, as_, bc, bs, dtype=dt)
    for stride in (n, n + 3):     # results side by side, and with room between the rows
        room = Room(m * stride * dt.itemsize)
        assert load().AnnB200MatmulBlocks(a.ptr, pad, sa.ptr, 0, b.ptr, pad, sb.ptr, int(square), m, n, k, types[out],
                                          room.ptr, stride, st) == 0
        torch.cuda.synchronize()
        got = room.view(dt, (m, stride))
        assert room.guards_are_whole() and torch.equal(got[:, :n], want)
        assert bool((got[:, n:].contiguous().view(torch.uint8) == 0xff).all())


@pytest.mark.parametrize('dtype', ['float32', 'float16', 'bfloat16'])
@pytest.mark.parametrize('nq', [40, 200])
@pytest.mark.parametrize('dims', [1, 3, 77, 130])
def test_what_lies_between_the_rows_does_not_count(cuda, dtype, nq, dims):
    # rows on 16-byte boundaries that end off them, NaN up to the next one
    import torch
    import pgvector_b200 as pb
    dt = getattr(torch, dtype)
    g = torch.Generator(device='cuda')
    g.manual_seed(dims)
    x = torch.randn((nq, dims), generator=g, device='cuda').to(dt)
    w = torch.randn((900, dims), generator=g, device='cuda').to(dt)
    t = torch.randint(0, 900, (nq,), generator=g, device='cuda')
    pad = (dims + 7) // 8 * 8 + 8
    hx = torch.full((nq, pad), float('nan'), dtype=dt, device='cuda')
    hw = torch.full((900, pad), float('nan'), dtype=dt, device='cuda')
    hx[:, :dims], hw[:, :dims] = x, w
    loss, lse = pb.softmax_loss(x, w, t, scale=0.3)
    want = (loss, lse) + pb.softmax_loss_grad(x, w, t, lse, scale=0.3)
    for a, b in ((hx[:, :dims], hw[:, :dims]), (x, hw[:, :dims]), (hx[:, :dims], w)):
        loss, lse = pb.softmax_loss(a, b, t, scale=0.3)
        got = (loss, lse) + pb.softmax_loss_grad(a, b, t, lse, scale=0.3)
        for u, v in zip(got, want):
            assert torch.equal(u, v)
