"""The workspace question of the softmax loss."""
import ctypes

import pytest

import pgvector_b200 as pb
from pgvector_b200._lib import load
from test_ops_cpu import FAKE, loss_job


def sizes(job):
    a, b = ctypes.c_uint64(), ctypes.c_uint64()
    assert load().AnnB200SoftmaxLossWorkspace(ctypes.byref(job), ctypes.byref(a), ctypes.byref(b)) == pb.OK
    return a.value, b.value


@pytest.mark.parametrize('dtype', [pb.F32, pb.F16, pb.BF16])
def test_pointers_set_later_do_not_change_it(dtype):
    """The job's sizes, types, strides and operands decide; outputs and weights may be set after the question."""
    full = sizes(loss_job(dtype=dtype, grad=FAKE))
    assert sizes(loss_job(dtype=dtype, grad=None)) == full
    assert sizes(loss_job(dtype=dtype, grad=FAKE, dqueries=None)) == full
    assert sizes(loss_job(dtype=dtype, grad=None, loss=None, lse=None, drows=None, workspace=None)) == full
