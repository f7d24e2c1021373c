"""Training and low-precision products over a shard's rows (CUDA tensors in and
out; the kernels are libannb200.so's, see annb200.h for the exact terms).

  * ``softmax_loss`` / ``softmax_loss_grad`` - cross entropy of queries with all
    rows as classes, without keeping the logits, and its gradients.
  * ``quantize_blocks`` - E4M3 codes with one FP32 scale per block of 128.
  * ``matmul_blocks`` - the product of two operands in that form.

Calls enqueue their work on ``stream`` (default: torch's current stream of the
operands' device) and return at once. Their outputs and workspace are
allocated for that stream, so they can be captured into a CUDA graph. Bad
arguments raise AnnB200Error (ANN_INVALID). softmax_loss takes part in autograd;
codes, scales and products of codes are not differentiable and never require a
gradient.
"""
import contextlib
import ctypes
import functools

from . import _abi
from ._lib import AnnB200Error, INVALID, check, load

BLOCK = 128
# torch, its types' numbers in annb200.h and those of E4M3 codes: from the first
# call on (the package and its names are there without torch)
torch, TYPES, E4M3 = None, {}, ()


def _with_torch():
    global torch, TYPES, E4M3
    if torch is None:
        import torch as module
        TYPES = {module.float32: 0, module.float16: 1, module.bfloat16: 5}
        E4M3 = (module.float8_e4m3fn, module.uint8)
        torch = module


def _need(ok, message, *args):
    if not ok:
        raise AnnB200Error(INVALID, message % args)


def _matrix(t, name, dtypes, like=None):
    """A CUDA matrix whose rows are contiguous; its row stride in elements."""
    if not (isinstance(t, torch.Tensor) and t.dim() == 2 and t.dtype in dtypes and t.is_cuda):
        _need(isinstance(t, torch.Tensor) and t.dim() == 2, '%s: not a matrix', name)
        _need(t.dtype in dtypes, '%s: type %s', name, t.dtype)
        _need(False, '%s: not a CUDA tensor', name)
    _need(like is None or t.device == like.device, '%s: on another device', name)
    m, n = t.shape
    stride, inner = t.stride()
    _need(n <= 1 or inner == 1, '%s: its rows are not contiguous', name)
    if m <= 1:
        return max(stride, n)
    _need(stride >= n, '%s: its rows overlap', name)
    return stride


def _vector(t, name, n, dtype, like):
    _need(isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == (n,) and t.device == like.device
          and t.is_contiguous(), '%s: not a contiguous %s [%d] on the operands\' device', name, dtype, n)
    return t.data_ptr()


@contextlib.contextmanager
def _elsewhere(device, stream, tensors):
    with torch.cuda.device(device):
        current = torch.cuda.current_stream(device)
        if stream is None or stream == current:
            yield current.cuda_stream
            return
        _need(stream.device == device, 'the stream is of another device')
        with torch.cuda.stream(stream):
            yield stream.cuda_stream
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _run(stream, tensors, call):
    """call(raw stream) with the operands' device current and, where one is given,
    `stream` as torch's: what call allocates belongs to it, and operands made on
    another stream are kept from reuse until its work is done."""
    device = tensors[0].device
    if stream is None and torch.cuda.current_device() == device.index:
        return call(torch._C._cuda_getCurrentRawStream(device.index))
    with _elsewhere(device, stream, tensors) as st:
        return call(st)


def _loss_job(queries, rows, targets, scale):
    row_stride = _matrix(rows, 'rows', TYPES)
    query_stride = _matrix(queries, 'queries', (rows.dtype,), rows)
    nq, dims = queries.shape
    _need(dims == rows.shape[1], 'queries of %d dimensions, rows of %d', dims, rows.shape[1])
    return _abi.AnnB200LossJob(
        TYPES[rows.dtype], dims, nq, float(scale), rows.shape[0], queries.data_ptr(), query_stride, rows.data_ptr(),
        row_stride, _vector(targets, 'targets', nq, torch.int64, rows))


def _workspace(job, which, device):
    """Room for the call, held by the tensor that is returned."""
    need = (ctypes.c_uint64(), ctypes.c_uint64())
    check(load().AnnB200SoftmaxLossWorkspace(ctypes.byref(job), ctypes.byref(need[0]), ctypes.byref(need[1])))
    size = need[which].value
    ws = torch.empty((size,), dtype=torch.uint8, device=device)
    job.workspace, job.workspace_bytes = ws.data_ptr(), size
    return ws


def softmax_loss(queries, rows, targets, scale=1.0, status=None, stream=None):
    """Cross entropy of each query with all `rows` as the classes:
    lse_i - scale * <query_i, row_targets[i]>, lse_i = log sum_j exp(scale *
    <query_i, row_j>). queries [nq, dims] and rows [n, dims] of one type
    (float32, float16, bfloat16); targets int64 [nq], negative for none (loss
    0). status: optional int32 [nq], ANN_INVALID for a target >= n (loss NaN).
    Returns (loss, lse), float32 [nq].

    Where queries or rows require a gradient, so does the loss: its backward pass
    is softmax_loss_grad, once. lse has no gradient of its own: a backward pass
    that reaches it raises AnnB200Error. (As with all of torch's operators, a
    backward pass is captured into a CUDA graph only while no graph of the same
    leaves made outside of the capture is alive.)"""
    _with_torch()
    job = _loss_job(queries, rows, targets, scale)
    if status is not None:
        job.status = _vector(status, 'status', queries.shape[0], torch.int32, rows)
    if (queries.requires_grad or rows.requires_grad) and torch.is_grad_enabled():
        return _run(stream, (queries, rows, targets, status),
                    lambda st: _autograd().apply(queries, rows, targets, job))
    return _run(stream, (queries, rows, targets, status),
                lambda st: _enqueue_loss(job, rows.device, st,
                                         torch.empty((2, job.nq), dtype=torch.float32, device=rows.device).unbind()))


def _enqueue_loss(job, device, st, out):
    job.loss, job.lse = out[0].data_ptr(), out[1].data_ptr()
    ws = _workspace(job, 0, device)  # noqa: F841
    check(load().AnnB200SoftmaxLoss(ctypes.byref(job), st))
    return out


@functools.cache
def _autograd():
    class SoftmaxLoss(torch.autograd.Function):
        @staticmethod
        def forward(ctx, queries, rows, targets, job):
            # (on the stream that _run made current, and so is the backward pass)
            loss = torch.empty((job.nq,), dtype=torch.float32, device=rows.device)
            lse = torch.empty_like(loss)
            _enqueue_loss(job, rows.device, torch._C._cuda_getCurrentRawStream(rows.device.index), (loss, lse))
            ctx.save_for_backward(queries, rows, targets, lse)
            ctx.set_materialize_grads(False)
            ctx.scale = job.scale
            return loss, lse

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, grad, grad_lse):
            _need(grad_lse is None, 'softmax_loss: lse has no gradient (detach it)')
            if grad is None:
                return None, None, None, None
            queries, rows, targets, lse = ctx.saved_tensors
            dq, dr = softmax_loss_grad(queries, rows, targets, lse, grad=grad.contiguous(), scale=ctx.scale,
                                       need_queries=ctx.needs_input_grad[0], need_rows=ctx.needs_input_grad[1])
            return dq, dr, None, None

    return SoftmaxLoss


def softmax_loss_grad(queries, rows, targets, lse, grad=None, scale=1.0, need_queries=True, need_rows=True,
                      stream=None):
    """Gradients of sum_i grad_i * loss_i by the queries and the rows, from the
    inputs of softmax_loss and the lse it returned for them (no other: one joined
    over several calls' rows gives wrong dqueries). grad: float32 [nq], by
    default ones. Returns (dqueries, drows) of the operands' type; None for one
    that is not needed. They are not differentiable further. softmax_loss calls
    this in its backward pass; by hand, ``queries.backward(dqueries)``."""
    _with_torch()
    job = _loss_job(queries, rows, targets, scale)
    nq, device = queries.shape[0], rows.device
    job.lse = _vector(lse, 'lse', nq, torch.float32, rows)
    if grad is not None:
        job.grad = _vector(grad, 'grad', nq, torch.float32, rows)

    def call(st):
        dq = torch.empty(queries.shape, dtype=rows.dtype, device=device) if need_queries else None
        dr = torch.empty(rows.shape, dtype=rows.dtype, device=device) if need_rows else None
        if need_queries:
            job.dqueries = dq.data_ptr()
        if need_rows:
            job.drows = dr.data_ptr()
            if nq == 0:
                dr.zero_()
        ws = _workspace(job, 1, device)  # noqa: F841
        check(load().AnnB200SoftmaxLossGrad(ctypes.byref(job), st))
        return dq, dr

    return _run(stream, (queries, rows, targets, lse, grad), call)


def quantize_blocks(x, square=False, stream=None):
    """E4M3 codes of x [m, k] (float32, float16, bfloat16) with one FP32 scale
    per 1 x 128 block of a row, or per 128 x 128 block (square). Returns
    (codes float8_e4m3fn [m, k], a view of rows of a multiple of 16 bytes;
    scales float32 [m or ceil(m/128), ceil(k/128)])."""
    _with_torch()
    stride = _matrix(x, 'x', TYPES)
    m, k = x.shape
    pad = (k + 15) // 16 * 16

    def call(st):
        codes = torch.empty((m, pad), dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty(((m + BLOCK - 1) // BLOCK if square else m, (k + BLOCK - 1) // BLOCK),
                             dtype=torch.float32, device=x.device)
        check(load().AnnB200QuantizeBlocks(TYPES[x.dtype], x.data_ptr(), stride, m, k, int(bool(square)),
                                           codes.data_ptr(), pad, scales.data_ptr(), st))
        return codes if pad == k else codes[:, :k], scales

    return _run(stream, (x,), call)


def _operand(codes, scales, name, like=None):
    """(row stride in bytes, whether its blocks are square) of an E4M3 operand."""
    stride = _matrix(codes, name, E4M3, like)
    m, k = codes.shape
    if m <= 1:
        stride = (stride + 15) // 16 * 16
    kb, tall = (k + BLOCK - 1) // BLOCK, (m + BLOCK - 1) // BLOCK
    _need(isinstance(scales, torch.Tensor) and scales.dtype == torch.float32 and scales.device == codes.device
          and scales.is_contiguous() and scales.shape in ((m, kb), (tall, kb)),
          '%s: scales are not a contiguous float32 [%d or %d, %d] on its device', name, m, tall, kb)
    return stride, int(scales.shape[0] != m)


def matmul_blocks(a, a_scales, b, b_scales, dtype=None, stream=None):
    """out[i][j] = sum over blocks of 128 of a_scale * b_scale * <a_i, b_j>: the
    scores of a's rows against b's, of operands as quantize_blocks makes them
    (rows a multiple of 16 bytes apart, 16-byte aligned). Each side's scales
    have one row per row, or one per 128 rows (square blocks). dtype: float32
    (default), float16 or bfloat16. Returns [m, n]."""
    _with_torch()
    dtype = dtype or torch.float32
    _need(dtype in TYPES, 'output type %s', dtype)
    sa, qa = _operand(a, a_scales, 'a')
    sb, qb = _operand(b, b_scales, 'b', a)
    m, k = a.shape
    n = b.shape[0]
    _need(k == b.shape[1], 'a has %d columns, b %d', k, b.shape[1])

    def call(st):
        out = torch.empty((m, n), dtype=dtype, device=a.device)
        check(load().AnnB200MatmulBlocks(a.data_ptr(), sa, a_scales.data_ptr(), qa, b.data_ptr(), sb,
                                         b_scales.data_ptr(), qb, m, n, k, TYPES[dtype], out.data_ptr(), n, st))
        return out

    return _run(stream, (a, a_scales, b, b_scales), call)
