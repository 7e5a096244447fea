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

_F32 = torch.float32
_current_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)  # without the lazy-init check
_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


# A call on a few rows costs what its checks cost (a launch is 2.5 us of host time): each reads a tensor's attributes once.
def _rows(t, shape, name):
    """(rows, row stride in elements) of a tensor of this shape whose last axis is contiguous."""
    strides = t.stride()
    if len(strides) == 2 and strides[1] == 1 and shape[1]:
        return shape[0], strides[0]
    if not strides or shape[-1] == 0:
        raise ValueError('%s: at least one axis and one entry per row expected, got %s' % (name, tuple(shape)))
    n = shape[-1]
    if n > 1 and strides[-1] != 1:
        raise ValueError('%s: the last axis must be contiguous (strides %s)' % (name, strides))
    if t.is_contiguous():
        return t.numel() // n, n
    rows, ld = 1, n
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size == 1:
            continue
        if rows == 1:
            ld = stride
        elif stride != rows * ld:
            raise ValueError('%s: its rows do not lie one stride apart (shape %s, strides %s)' % (name, tuple(shape), strides))
        rows *= size
    return rows, ld


def _input(x):
    """(dtype, its code, device index, shape) of the matrix."""
    dtype, device = x.dtype, x.get_device()
    code = _DTYPE.get(dtype)
    if code is None:
        raise ValueError('layer norm takes float32, bfloat16 or float16, got %s' % dtype)
    if device < 0 or device != _current_device():
        raise ValueError('layer norm runs on the current device, got a tensor on %s' % x.device)
    return dtype, code, device, x.shape


def _like(t, name, device, dtype, shape):
    """Row stride of a matrix that must be like x."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device:
        raise ValueError('%s: %s %s on cuda:%d expected, got %s %s on %s' % (name, dtype, tuple(shape), device, t.dtype, tuple(t.shape), t.device))
    return _rows(t, shape, name)[1]


def _weight(w, name, dtype, n, device, code):
    """dtype code of a weight vector; code: what the others have, None so far."""
    t = w.dtype
    got = _DTYPE[t] if t is _F32 or t is dtype else None
    if got is None or w.shape != (n,) or not w.is_contiguous() or w.get_device() != device:
        raise ValueError('%s: %d contiguous entries of float32 or %s on cuda:%d expected, got %s %s on %s'
                         % (name, n, dtype, device, t, tuple(w.shape), w.device))
    if code is not None and got != code:
        raise ValueError('%s: the weight vectors must share one type' % name)
    return got


def _stats(stats, shape, device):
    want = (shape[0], 2) if len(shape) == 2 else shape[:-1] + (2,)
    if stats.dtype is not _F32 or stats.shape != want or not stats.is_contiguous() or stats.get_device() != device:
        raise ValueError('stats: contiguous float32 %s on cuda:%d expected, got %s %s on %s'
                         % (tuple(shape[:-1]) + (2,), device, stats.dtype, tuple(stats.shape), stats.device))


def layer_norm(x, gamma=None, beta=None, eps=LN_EPS, out=None, stats=None):
    """-> (out, stats): out = (x - mean) * rstd * gamma + beta over the last axis, stats[..., 0:2] = (mean, rstd) in float32
    (the layout of ``feature_row_stats``).  ``out`` may be x itself or other columns of the table x is a slice of; no other
    argument may share memory with ``out`` or ``stats``, which are allocated when not given."""
    dtype, code, device, shape = _input(x)
    m, ldx = _rows(x, shape, 'x')
    n = shape[-1]
    w = g = b = None
    if gamma is not None:
        w = _weight(gamma, 'gamma', dtype, n, device, None)
        g = gamma.data_ptr()
    if beta is not None:
        w = _weight(beta, 'beta', dtype, n, device, w)
        b = beta.data_ptr()
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=x.device)
        ldy = n
    else:
        ldy = _like(out, 'out', device, dtype, shape)
    if stats is None:
        stats = torch.empty(shape[:-1] + (2,), dtype=_F32, device=x.device)
    else:
        _stats(stats, shape, device)
    rc = (_lib._lib or _lib.lib()).ultr_layer_norm_forward(
        x.data_ptr(), ldx, g, b, m, n, eps, code, w or 0, out.data_ptr(), ldy, stats.data_ptr(), _lib.stream_of(device))
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
    d_gamma / d_beta have gamma's type (float32 without gamma) unless given.  What is written (the workspace
    too) must not share memory with another argument; d_x may be other columns of the table that x or d_out is a slice of."""
    dtype, code, device, shape = _input(x)
    m, ldx = _rows(x, shape, 'x')
    n = shape[-1]
    lddy = _like(d_out, 'd_out', device, dtype, shape)
    _stats(stats, shape, device)
    need_x, need_g, need_b = need
    lib = _lib._lib or _lib.lib()
    w = g = px = pg = pb = ws = None
    lddx = n
    if gamma is not None:
        w = _weight(gamma, 'gamma', dtype, n, device, None)
        g = gamma.data_ptr()
    if need_g and d_gamma is not None:
        w = _weight(d_gamma, 'd_gamma', dtype, n, device, w)
    if need_b and d_beta is not None:
        w = _weight(d_beta, 'd_beta', dtype, n, device, w)
    w_dtype = dtype if w else _F32
    if not need_x:
        d_x = None
    else:
        if d_x is None:
            d_x = torch.empty(shape, dtype=dtype, device=x.device)
        else:
            lddx = _like(d_x, 'd_x', device, dtype, shape)
        px = d_x.data_ptr()
    if not need_g:
        d_gamma = None
    else:
        if d_gamma is None:
            d_gamma = torch.empty(n, dtype=w_dtype, device=x.device)
        pg = d_gamma.data_ptr()
    if not need_b:
        d_beta = None
    else:
        if d_beta is None:
            d_beta = torch.empty(n, dtype=w_dtype, device=x.device)
        pb = d_beta.data_ptr()
    nbytes = lib.ultr_layer_norm_workspace_bytes(m, n)
    if nbytes > 0:
        if workspace is None:
            workspace = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        elif workspace.numel() * workspace.element_size() < nbytes or not workspace.is_contiguous() or workspace.get_device() != device:
            raise ValueError('workspace: layer_norm_workspace(%d, %d, %s) expected' % (m, n, x.device))
        ws = workspace.data_ptr()
    rc = lib.ultr_layer_norm_backward(d_out.data_ptr(), lddy, x.data_ptr(), ldx, stats.data_ptr(), g, m, n, code, w or 0, px, lddx,
                                      pg, pb, ws, _lib.stream_of(device))
    if rc:
        _lib.check(rc, 'ultr_layer_norm_backward')
    return d_x, d_gamma, d_beta
