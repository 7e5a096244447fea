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


def _rows(t, name):
    """(rows, row stride in elements) of a tensor whose last axis is contiguous."""
    n = t.shape[-1] if t.dim() else 0
    if t.dim() == 0 or n == 0:
        raise ValueError('%s: at least one axis and one entry per row expected, got %s' % (name, tuple(t.shape)))
    if n > 1 and t.stride(-1) != 1:
        raise ValueError('%s: the last axis must be contiguous (strides %s)' % (name, t.stride()))
    if t.dim() == 2:
        return t.shape[0], t.stride(0)
    if t.is_contiguous():
        return t.numel() // n, n
    rows, ld = 1, n
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if rows == 1:
            ld = stride
        elif stride != rows * ld:
            raise ValueError('%s: its rows do not lie one stride apart (shape %s, strides %s)' % (name, tuple(t.shape), t.stride()))
        rows *= size
    return rows, ld


def _check(t, name, device, dtype, shape):
    if t.device != device or t.dtype != dtype or t.shape != shape:
        raise ValueError('%s: %s %s on %s expected, got %s %s on %s' % (name, dtype, tuple(shape), device, t.dtype, tuple(t.shape), t.device))


def _input(x):
    dtype = _DTYPE.get(x.dtype)
    if dtype is None:
        raise ValueError('layer norm takes float32, bfloat16 or float16, got %s' % x.dtype)
    if not x.is_cuda or x.device.index != torch.cuda.current_device():
        raise ValueError('layer norm runs on the current device (cuda:%s), got a tensor on %s'
                         % (torch.cuda.current_device() if torch.cuda.is_available() else '-', x.device))
    return dtype


def _weight(w, name, x, w_dtype):
    """dtype code of a weight vector (None: keeps what the others have)."""
    if w is None:
        return w_dtype
    if w.dtype != torch.float32 and w.dtype != x.dtype:
        raise ValueError('%s: float32 or %s expected, got %s' % (name, x.dtype, w.dtype))
    _check(w, name, x.device, w.dtype, x.shape[-1:])
    if not w.is_contiguous():
        raise ValueError('%s must be contiguous' % name)
    code = _DTYPE[w.dtype]
    if w_dtype is not None and code != w_dtype:
        raise ValueError('%s: the weight vectors must share one type' % name)
    return code


def _stats(stats, x):
    _check(stats, 'stats', x.device, torch.float32, x.shape[:-1] + (2,))
    if not stats.is_contiguous():
        raise ValueError('stats must be contiguous')


def layer_norm(x, gamma=None, beta=None, eps=LN_EPS, out=None, stats=None):
    """-> (out, stats): out = (x - mean) * rstd * gamma + beta over the last axis, stats[..., 0:2] = (mean, rstd) in float32
    (the layout of ``feature_row_stats``).  ``out`` may be x itself; ``out`` / ``stats`` are allocated when not given."""
    code = _input(x)
    m, ldx = _rows(x, 'x')
    w = _weight(beta, 'beta', x, _weight(gamma, 'gamma', x, None))
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _check(out, 'out', x.device, x.dtype, x.shape)
    my, ldy = _rows(out, 'out')
    if stats is None:
        stats = torch.empty(x.shape[:-1] + (2,), dtype=torch.float32, device=x.device)
    else:
        _stats(stats, x)
    _lib.check(_lib.lib().ultr_layer_norm_forward(
        x.data_ptr(), ldx, None if gamma is None else gamma.data_ptr(), None if beta is None else beta.data_ptr(), m,
        x.shape[-1], eps, code, _lib.DTYPE_F32 if w is None else w, out.data_ptr(), ldy, stats.data_ptr(),
        _lib.current_stream()), 'ultr_layer_norm_forward')
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
    code = _input(x)
    m, ldx = _rows(x, 'x')
    _check(d_out, 'd_out', x.device, x.dtype, x.shape)
    _, lddy = _rows(d_out, 'd_out')
    _stats(stats, x)
    w = _weight(gamma, 'gamma', x, None)
    need_x, need_g, need_b = need
    wdt = torch.float32 if gamma is None else gamma.dtype
    lddx = 0
    if need_x:
        if d_x is None:
            d_x = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        else:
            _check(d_x, 'd_x', x.device, x.dtype, x.shape)
        _, lddx = _rows(d_x, 'd_x')
    if need_g:
        if d_gamma is None:
            d_gamma = torch.empty(x.shape[-1:], dtype=wdt, device=x.device)
        else:
            w = _weight(d_gamma, 'd_gamma', x, w)
    if need_b:
        if d_beta is None:
            d_beta = torch.empty(x.shape[-1:], dtype=wdt if d_gamma is None or not need_g else d_gamma.dtype, device=x.device)
        w = _weight(d_beta, 'd_beta', x, w)
    if need_g:
        w = _weight(d_gamma, 'd_gamma', x, w)
    ws = None
    n = x.shape[-1]
    if need_g or need_b or n > 8192:
        if workspace is None:
            workspace = layer_norm_workspace(m, n, x.device)
        elif workspace.device != x.device or not workspace.is_contiguous() or \
                workspace.numel() * workspace.element_size() < _lib.lib().ultr_layer_norm_workspace_bytes(m, n):
            raise ValueError('workspace: layer_norm_workspace(%d, %d, %s) expected' % (m, n, x.device))
        ws = workspace.data_ptr() or None
    _lib.check(_lib.lib().ultr_layer_norm_backward(
        d_out.data_ptr(), lddy, x.data_ptr(), ldx, stats.data_ptr(), None if gamma is None else gamma.data_ptr(), m,
        x.shape[-1], code, _lib.DTYPE_F32 if w is None else w, d_x.data_ptr() if need_x else None, lddx,
        d_gamma.data_ptr() if need_g else None, d_beta.data_ptr() if need_b else None, ws, _lib.current_stream()),
        'ultr_layer_norm_backward')
    return d_x if need_x else None, d_gamma if need_g else None, d_beta if need_b else None
