"""Training and low-precision products over a shard's rows (CUDA tensors in and
out; the kernels are libannb200.so's, see annb200.h for the exact terms).

  * ``softmax_loss`` / ``softmax_loss_grad`` - cross entropy of queries with all
    rows as classes, without keeping the logits, and its gradients.
  * ``quantize_blocks`` - E4M3 codes with one FP32 scale per block of 128.
  * ``matmul_blocks`` - the product of two operands in that form.

Calls enqueue their work on ``stream`` (default: torch's current stream of the
operands' device) and return at once. Their outputs and workspace are
allocated for that stream, so they can be captured into a CUDA graph. Bad
arguments raise AnnB200Error (ANN_INVALID).
"""
import contextlib
import ctypes

from . import _abi
from ._lib import AnnB200Error, INVALID, check, load

BLOCK = 128


def _types():
    import torch
    return {torch.float32: 0, torch.float16: 1, torch.bfloat16: 5}


def _need(ok, message, *args):
    if not ok:
        raise AnnB200Error(INVALID, message % args)


def _matrix(t, name, dtypes, like=None):
    """A CUDA matrix whose rows are contiguous; its row stride in elements."""
    import torch
    _need(isinstance(t, torch.Tensor) and t.dim() == 2, '%s: not a matrix', name)
    _need(t.dtype in dtypes, '%s: type %s', name, t.dtype)
    _need(t.is_cuda, '%s: not a CUDA tensor', name)
    _need(like is None or t.device == like.device, '%s: on another device', name)
    _need(t.shape[1] <= 1 or t.stride(1) == 1, '%s: its rows are not contiguous', name)
    if t.shape[0] <= 1:
        return max(t.stride(0), t.shape[1])
    _need(t.stride(0) >= t.shape[1], '%s: its rows overlap', name)
    return t.stride(0)


def _vector(t, name, n, dtype, like):
    import torch
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype and tuple(t.shape) == (n,) and t.device == like.device
          and t.is_contiguous(), '%s: not a contiguous %s [%d] on the operands\' device', name, dtype, n)
    return t.data_ptr()


@contextlib.contextmanager
def _call(stream, *tensors):
    """The operands' device made current, and `stream` where one is given: what
    is allocated inside belongs to it, and operands made on another stream are
    kept from reuse until its work is done."""
    import torch
    device = tensors[0].device
    with torch.cuda.device(device):
        current = torch.cuda.current_stream(device)
        if stream is None or stream == current:
            yield ctypes.c_void_p(current.cuda_stream)
            return
        _need(stream.device == device, 'the stream is of another device')
        with torch.cuda.stream(stream):
            yield ctypes.c_void_p(stream.cuda_stream)
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _loss_job(queries, rows, targets, scale):
    import torch
    types = _types()
    job = _abi.AnnB200LossJob()
    job.row_stride = _matrix(rows, 'rows', types)
    job.query_stride = _matrix(queries, 'queries', (rows.dtype,), rows)
    _need(queries.shape[1] == rows.shape[1], 'queries of %d dimensions, rows of %d', queries.shape[1], rows.shape[1])
    job.dtype, job.dims, job.nq, job.nrows = types[rows.dtype], rows.shape[1], queries.shape[0], rows.shape[0]
    job.scale = float(scale)
    job.queries, job.rows = queries.data_ptr(), rows.data_ptr()
    job.targets = _vector(targets, 'targets', queries.shape[0], torch.int64, rows)
    return job


def _run_loss(fn, which, job, device, st):
    import torch
    need = (ctypes.c_uint64(), ctypes.c_uint64())
    check(load().AnnB200SoftmaxLossWorkspace(ctypes.byref(job), ctypes.byref(need[0]), ctypes.byref(need[1])))
    ws = torch.empty((max(need[which].value, 1),), dtype=torch.uint8, device=device)
    job.workspace, job.workspace_bytes = ws.data_ptr(), ws.numel()
    check(fn(ctypes.byref(job), st))


def softmax_loss(queries, rows, targets, scale=1.0, status=None, stream=None):
    """Cross entropy of each query with all `rows` as the classes:
    lse_i - scale * <query_i, row_targets[i]>, lse_i = log sum_j exp(scale *
    <query_i, row_j>). queries [nq, dims] and rows [n, dims] of one type
    (float32, float16, bfloat16); targets int64 [nq], negative for none (loss
    0). status: optional int32 [nq], ANN_INVALID for a target >= n (loss NaN).
    Returns (loss, lse), float32 [nq]."""
    import torch
    job = _loss_job(queries, rows, targets, scale)
    if status is not None:
        job.status = _vector(status, 'status', queries.shape[0], torch.int32, rows)
    with _call(stream, queries, rows, targets, status) as st:
        loss = torch.empty((queries.shape[0],), dtype=torch.float32, device=rows.device)
        lse = torch.empty_like(loss)
        job.loss, job.lse = loss.data_ptr(), lse.data_ptr()
        _run_loss(load().AnnB200SoftmaxLoss, 0, job, rows.device, st)
    return loss, lse


def softmax_loss_grad(queries, rows, targets, lse, grad=None, scale=1.0, need_queries=True, need_rows=True,
                      stream=None):
    """Gradients of sum_i grad_i * loss_i by the queries and the rows, from the
    inputs of softmax_loss and the lse it returned. grad: float32 [nq], by
    default ones. Returns (dqueries, drows) of the operands' type; None for one
    that is not needed. With torch.autograd in the encoder:
    ``queries.backward(dqueries)``."""
    import torch
    job = _loss_job(queries, rows, targets, scale)
    job.lse = _vector(lse, 'lse', queries.shape[0], torch.float32, rows)
    if grad is not None:
        job.grad = _vector(grad, 'grad', queries.shape[0], torch.float32, rows)
    with _call(stream, queries, rows, targets, lse, grad) as st:
        dq = torch.empty(queries.shape, dtype=rows.dtype, device=rows.device) if need_queries else None
        dr = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device) if need_rows else None
        job.dqueries = dq.data_ptr() if need_queries else None
        job.drows = dr.data_ptr() if need_rows else None
        if queries.shape[0] == 0 and need_rows:
            dr.zero_()
        _run_loss(load().AnnB200SoftmaxLossGrad, 1, job, rows.device, st)
    return dq, dr


def quantize_blocks(x, square=False, stream=None):
    """E4M3 codes of x [m, k] (float32, float16, bfloat16) with one FP32 scale
    per 1 x 128 block of a row, or per 128 x 128 block (square). Returns
    (codes float8_e4m3fn [m, k], a view of rows of a multiple of 16 bytes;
    scales float32 [m or ceil(m/128), ceil(k/128)])."""
    import torch
    stride = _matrix(x, 'x', _types())
    m, k = x.shape
    with _call(stream, x) as st:
        codes = torch.empty((m, (k + 15) // 16 * 16), dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty(((m + BLOCK - 1) // BLOCK if square else m, (k + BLOCK - 1) // BLOCK),
                             dtype=torch.float32, device=x.device)
        check(load().AnnB200QuantizeBlocks(_types()[x.dtype], x.data_ptr(), stride, m, k, int(bool(square)),
                                           codes.data_ptr(), codes.shape[1], scales.data_ptr(), st))
    return codes[:, :k], scales


def _operand(codes, scales, name, like=None):
    """(row stride in bytes, whether its blocks are square) of an E4M3 operand."""
    import torch
    stride = _matrix(codes, name, (torch.float8_e4m3fn, torch.uint8), like)
    if codes.shape[0] <= 1:
        stride = (stride + 15) // 16 * 16
    m, kb = codes.shape[0], (codes.shape[1] + BLOCK - 1) // BLOCK
    _need(isinstance(scales, torch.Tensor) and scales.dtype == torch.float32 and scales.device == codes.device
          and scales.is_contiguous() and tuple(scales.shape) in ((m, kb), ((m + BLOCK - 1) // BLOCK, kb)),
          '%s: scales are not a contiguous float32 [%d or %d, %d] on its device', name, m, (m + BLOCK - 1) // BLOCK, kb)
    return stride, int(scales.shape[0] != m)


def matmul_blocks(a, a_scales, b, b_scales, dtype=None, stream=None):
    """out[i][j] = sum over blocks of 128 of a_scale * b_scale * <a_i, b_j>: the
    scores of a's rows against b's, of operands as quantize_blocks makes them
    (rows a multiple of 16 bytes apart, 16-byte aligned). Each side's scales
    have one row per row, or one per 128 rows (square blocks). dtype: float32
    (default), float16 or bfloat16. Returns [m, n]."""
    import torch
    dtype = dtype or torch.float32
    _need(dtype in _types(), 'output type %s', dtype)
    sa, qa = _operand(a, a_scales, 'a')
    sb, qb = _operand(b, b_scales, 'b', a)
    _need(a.shape[1] == b.shape[1], 'a has %d columns, b %d', a.shape[1], b.shape[1])
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    with _call(stream, a, a_scales, b, b_scales) as st:
        out = torch.empty((m, n), dtype=dtype, device=a.device)
        check(load().AnnB200MatmulBlocks(a.data_ptr(), sa, a_scales.data_ptr(), qa, b.data_ptr(), sb,
                                         b_scales.data_ptr(), qb, m, n, k, _types()[dtype], out.data_ptr(), n, st))
    return out
