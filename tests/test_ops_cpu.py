"""Refusals of the operator calls, checked on the host before any device work."""
import ctypes

import pytest

import pgvector_b200 as pb
from pgvector_b200 import _abi
from pgvector_b200._lib import load

FAKE = 4096   # an aligned address that is never read


def loss_job(**over):
    job = _abi.AnnB200LossJob()
    d = dict(dtype=pb.F32, dims=8, nq=4, scale=1.0, nrows=16, queries=FAKE, query_stride=8, rows=FAKE, row_stride=8,
             targets=FAKE, loss=FAKE, lse=FAKE, dqueries=FAKE, drows=FAKE, workspace=FAKE, workspace_bytes=1 << 40)
    d.update(over)
    for k, v in d.items():
        setattr(job, k, v)
    return job


def call(fn, job):
    return getattr(load(), fn)(ctypes.byref(job), None)


@pytest.mark.parametrize('fn', ['AnnB200SoftmaxLoss', 'AnnB200SoftmaxLossGrad'])
@pytest.mark.parametrize('over', [
    dict(dtype=pb.E4M3), dict(dtype=pb.BIT), dict(dtype=99), dict(dims=0), dict(dims=65537), dict(nq=(1 << 22) + 1),
    dict(nrows=0), dict(nrows=1 << 31), dict(query_stride=7), dict(row_stride=7), dict(scale=float('inf')),
    dict(scale=float('nan')), dict(queries=None), dict(rows=None), dict(targets=None), dict(workspace=None),
    dict(workspace_bytes=0), dict(workspace=FAKE + 16)])
def test_loss_refusals(fn, over):
    assert call(fn, loss_job(**over)) == pb.INVALID
    assert load().AnnB200LastError()


def test_loss_calls_with_nothing_to_do():
    assert call('AnnB200SoftmaxLoss', loss_job(nq=0, queries=None, targets=None, workspace=None)) == pb.OK
    assert call('AnnB200SoftmaxLossGrad', loss_job(nq=0, queries=None, targets=None, workspace=None)) == pb.OK
    assert call('AnnB200SoftmaxLossGrad', loss_job(dqueries=None, drows=None, workspace=None)) == pb.OK
    assert call('AnnB200SoftmaxLossGrad', loss_job(lse=None)) == pb.INVALID
    assert load().AnnB200SoftmaxLoss(None, None) == pb.INVALID


@pytest.mark.parametrize('dtype', [pb.F32, pb.F16, pb.BF16])
@pytest.mark.parametrize('nq,nrows,dims', [(1, 1, 1), (4096, 65536, 768), (1, 0x7fffffff, 65536), (1 << 22, 1000, 8)])
def test_workspace_is_given_for_every_size(dtype, nq, nrows, dims):
    a, b = ctypes.c_uint64(), ctypes.c_uint64()
    job = loss_job(dtype=dtype, nq=nq, nrows=nrows, dims=dims, query_stride=dims, row_stride=dims)
    assert load().AnnB200SoftmaxLossWorkspace(ctypes.byref(job), ctypes.byref(a), ctypes.byref(b)) == pb.OK
    assert 0 < a.value and 0 < b.value
    assert load().AnnB200SoftmaxLossWorkspace(ctypes.byref(loss_job(dims=0)), None, None) == pb.INVALID


def quantize(**over):
    d = dict(dtype=pb.F32, x=FAKE, stride=128, m=4, k=128, square=0, codes=FAKE, code_stride=128, scales=FAKE)
    d.update(over)
    return load().AnnB200QuantizeBlocks(*d.values(), None)


@pytest.mark.parametrize('over', [
    dict(dtype=pb.E4M3), dict(dtype=77), dict(x=None), dict(codes=None), dict(scales=None), dict(stride=127),
    dict(code_stride=112), dict(code_stride=136), dict(codes=FAKE + 8), dict(m=1 << 31), dict(k=(1 << 20) + 1)])
def test_quantize_refusals(over):
    assert quantize(**over) == pb.INVALID


def test_quantize_with_nothing_to_do():
    assert quantize(m=0, x=None, codes=None, scales=None) == pb.OK
    assert quantize(k=0, x=None, codes=None, scales=None) == pb.OK


def matmul(**over):
    d = dict(a=FAKE, a_stride=128, a_scales=FAKE, a_square=0, b=FAKE, b_stride=128, b_scales=FAKE, b_square=0, m=4,
             n=8, k=128, out_dtype=pb.F32, out=FAKE, out_stride=8)
    d.update(over)
    return load().AnnB200MatmulBlocks(*d.values(), None)


@pytest.mark.parametrize('over', [
    dict(a=None), dict(b=None), dict(a_scales=None), dict(b_scales=None), dict(out=None), dict(a=FAKE + 8),
    dict(b=FAKE + 1), dict(a_stride=120), dict(a_stride=136), dict(b_stride=112), dict(out_stride=7),
    dict(out_dtype=pb.E4M3), dict(m=1 << 31), dict(n=1 << 31), dict(k=(1 << 20) + 1)])
def test_matmul_refusals(over):
    assert matmul(**over) == pb.INVALID


def test_matmul_with_nothing_to_do():
    assert matmul(m=0, a=None, out=None) == pb.OK
    assert matmul(n=0, b=None, out=None) == pb.OK


def test_python_refusals():
    import torch
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    bad = [
        lambda: pb.softmax_loss(x, x, t),                                   # not on a GPU
        lambda: pb.softmax_loss(x.double(), x.double(), t),
        lambda: pb.softmax_loss(x[0], x, t),
        lambda: pb.quantize_blocks(x),
        lambda: pb.quantize_blocks(x.to(torch.int32)),
        lambda: pb.matmul_blocks(x, x, x, x),
        lambda: pb.matmul_blocks(x.to(torch.float8_e4m3fn), x, x, x, dtype=torch.float64),
    ]
    for f in bad:
        with pytest.raises(pb.AnnB200Error) as e:
            f()
        assert e.value.status == pb.INVALID
