"""Layer normalisation of a tensor's rows as an operator of its own, forward and backward.

Reference: ultra/ranking_model/base_ranking_model.py:67-70 (NORM_FUNC_DIC['layer']), applied at DNN.py:78-81.  The DNN scorer
has it fused into its GEMMs; a ranking model that brings layers of its own calls these.  Like the scorer's passes they are
explicit (no autograd): ``layer_norm`` returns the row statistics, ``layer_norm_backward`` takes them.

Rows are the last axis, contiguous; the axes before it must be walkable with one stride (a row slice of a wider table is,
a transposed batch is not).  float32, bfloat16 and float16 tensors; gamma / beta in float32 or the tensor's type.  The calls
enqueue on torch's current stream of the current device, allocate nothing that the caller hands over, never synchronise, and
may be captured into a graph.
"""
import torch

from .. import _lib
from .DNN import LN_EPS

_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


# A call on a few rows costs what its checks cost: they use plain integer accessors, one pass over each tensor.
def _rows(t, name):
    """(rows, row stride in elements) of a tensor whose last axis is contiguous."""
    strides = t.stride()
    if not strides or t.shape[-1] == 0:
        raise ValueError('%s: at least one axis and one entry per row expected, got %s' % (name, tuple(t.shape)))
    n = t.shape[-1]
    if n > 1 and strides[-1] != 1:
        raise ValueError('%s: the last axis must be contiguous (strides %s)' % (name, strides))
    if len(strides) == 2:
        return t.shape[0], strides[0]
    if t.is_contiguous():
        return t.numel() // n, n
    rows, ld = 1, n
    for size, stride in zip(reversed(t.shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if rows == 1:
            ld = stride
        elif stride != rows * ld:
            raise ValueError('%s: its rows do not lie one stride apart (shape %s, strides %s)' % (name, tuple(t.shape), strides))
        rows *= size
    return rows, ld


def _input(x):
    """(dtype code, device index) of the matrix."""
    code, device = _DTYPE.get(x.dtype), x.get_device()
    if code is None:
        raise ValueError('layer norm takes float32, bfloat16 or float16, got %s' % x.dtype)
    if device < 0 or device != torch.cuda.current_device():
        raise ValueError('layer norm runs on the current device, got a tensor on %s' % x.device)
    return code, device


def _check(t, name, device, dtype, shape):
    if t.dtype != dtype or t.shape != shape or t.get_device() != device:
        raise ValueError('%s: %s %s on cuda:%d expected, got %s %s on %s' % (name, dtype, tuple(shape), device, t.dtype, tuple(t.shape), t.device))


def _weight(w, name, x, n, device, w_dtype):
    """dtype code of a weight vector; w_dtype: what the others have, None so far."""
    code = _DTYPE.get(w.dtype) if w.dtype == torch.float32 or w.dtype == x.dtype else None
    if code is None or w.dim() != 1 or w.numel() != n or not w.is_contiguous() or w.get_device() != device:
        raise ValueError('%s: %d contiguous entries of float32 or %s on cuda:%d expected, got %s %s on %s'
                         % (name, n, x.dtype, device, w.dtype, tuple(w.shape), w.device))
    if w_dtype is not None and code != w_dtype:
        raise ValueError('%s: the weight vectors must share one type' % name)
    return code


def _stats(stats, x, m, device):
    if stats.dtype != torch.float32 or stats.numel() != 2 * m or stats.shape[-1] != 2 or stats.dim() != x.dim() or \
            not stats.is_contiguous() or stats.get_device() != device or (x.dim() > 2 and stats.shape[:-1] != x.shape[:-1]):
        raise ValueError('stats: contiguous float32 %s on cuda:%d expected, got %s %s on %s'
                         % (tuple(x.shape[:-1]) + (2,), device, stats.dtype, tuple(stats.shape), stats.device))


def layer_norm(x, gamma=None, beta=None, eps=LN_EPS, out=None, stats=None):
    """-> (out, stats): out = (x - mean) * rstd * gamma + beta over the last axis, stats[..., 0:2] = (mean, rstd) in float32
    (the layout of ``feature_row_stats``).  ``out`` may be x itself; ``out`` / ``stats`` are allocated when not given."""
    code, device = _input(x)
    m, ldx = _rows(x, 'x')
    n = x.shape[-1]
    w = None
    if gamma is not None:
        w = _weight(gamma, 'gamma', x, n, device, w)
    if beta is not None:
        w = _weight(beta, 'beta', x, n, device, w)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out is not x:
        _check(out, 'out', device, x.dtype, x.shape)
    _, ldy = _rows(out, 'out')
    if stats is None:
        stats = torch.empty(x.shape[:-1] + (2,), dtype=torch.float32, device=x.device)
    else:
        _stats(stats, x, m, device)
    rc = _lib.lib().ultr_layer_norm_forward(
        x.data_ptr(), ldx, None if gamma is None else gamma.data_ptr(), None if beta is None else beta.data_ptr(), m, n, eps,
        code, _lib.DTYPE_F32 if w is None else w, out.data_ptr(), ldy, stats.data_ptr(), _lib.current_stream())
    if rc:
        _lib.check(rc, 'ultr_layer_norm_forward')
    return out, stats


def layer_norm_workspace(rows, width, device):
    """The workspace ``layer_norm_backward`` needs for ``rows`` rows of ``width`` entries.  One per call in flight: calls
    that share one (two streams, two captured graphs) must be ordered."""
    nbytes = _lib.lib().ultr_layer_norm_workspace_bytes(int(rows), int(width))
    if nbytes < 0:
        raise _lib.UltrError(_lib.lib().ultr_last_error().decode())
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def layer_norm_backward(d_out, x, stats, gamma=None, d_x=None, d_gamma=None, d_beta=None, workspace=None,
                        need=(True, True, True)):
    """-> (d_x, d_gamma, d_beta) for ``layer_norm(x, gamma, ...)`` that returned ``stats``.

    ``need``: which of the three are wanted; the others come back as None.  Gradients are written, not added to;
    d_gamma / d_beta have gamma's type (float32 without gamma) unless given.  d_x must not share memory with d_out or x."""
    code, device = _input(x)
    m, ldx = _rows(x, 'x')
    n = x.shape[-1]
    _check(d_out, 'd_out', device, x.dtype, x.shape)
    _, lddy = _rows(d_out, 'd_out')
    _stats(stats, x, m, device)
    need_x, need_g, need_b = need
    lib = _lib.lib()
    w = None
    if gamma is not None:
        w = _weight(gamma, 'gamma', x, n, device, w)
    if need_g and d_gamma is not None:
        w = _weight(d_gamma, 'd_gamma', x, n, device, w)
    if need_b and d_beta is not None:
        w = _weight(d_beta, 'd_beta', x, n, device, w)
    if w is None:
        w = _lib.DTYPE_F32
    w_dtype = torch.float32 if w == _lib.DTYPE_F32 else x.dtype
    lddx, ws = 0, None
    if not need_x:
        d_x = None
    else:
        if d_x is None:
            d_x = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _check(d_x, 'd_x', device, x.dtype, x.shape)
        _, lddx = _rows(d_x, 'd_x')
    if not need_g:
        d_gamma = None
    elif d_gamma is None:
        d_gamma = torch.empty(n, dtype=w_dtype, device=x.device)
    if not need_b:
        d_beta = None
    elif d_beta is None:
        d_beta = torch.empty(n, dtype=w_dtype, device=x.device)
    nbytes = lib.ultr_layer_norm_workspace_bytes(m, n)
    if nbytes > 0:
        if workspace is None:
            workspace = layer_norm_workspace(m, n, x.device)
        elif workspace.numel() * workspace.element_size() < nbytes or not workspace.is_contiguous() or workspace.get_device() != device:
            raise ValueError('workspace: layer_norm_workspace(%d, %d, %s) expected' % (m, n, x.device))
        ws = workspace.data_ptr()
    rc = lib.ultr_layer_norm_backward(
        d_out.data_ptr(), lddy, x.data_ptr(), ldx, stats.data_ptr(), None if gamma is None else gamma.data_ptr(), m, n, code, w,
        None if d_x is None else d_x.data_ptr(), lddx, None if d_gamma is None else d_gamma.data_ptr(),
        None if d_beta is None else d_beta.data_ptr(), ws, _lib.current_stream())
    if rc:
        _lib.check(rc, 'ultr_layer_norm_backward')
    return d_x, d_gamma, d_beta
