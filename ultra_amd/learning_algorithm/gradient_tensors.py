"""Global gradient norm, clipping and the Adagrad / SGD update over many separate tensors.

Reference: the clip by the global norm and the optimiser step over the list of trainable variables (dla.py:237-255,
ipw_rank.py:155-165).  The learning algorithms of this package keep their variables in one flat float32 buffer
(``ultr_clip_adagrad``); a model whose parameters are tensors of their own lists them here, once.
"""
import ctypes

import numpy as np
import torch

from .. import _lib
from ..ranking_model.DNN import parameters_written

_current_device = getattr(torch._C, '_cuda_getDevice', torch.cuda.current_device)  # without the lazy-init check
_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_REC = np.dtype([('grad', 'u8'), ('out', 'u8'), ('param', 'u8'), ('accum', 'u8'), ('copy', 'u8'), ('n', 'i8'),
                 ('grad_dtype', 'i4'), ('copy_dtype', 'i4')])  # _lib.UltrTensor, filled a column at a time
_STRATEGY = {'ada': _lib.OPT_ADAGRAD, 'sgd': _lib.OPT_SGD}  # the grad_strategy hparam


class GradientTensors(object):
    """A list of gradients (float32, bfloat16, float16, mixed as they come) and what belongs to them.

    grads    tensors of any shape, contiguous; a tensor without elements is allowed
    out      where ``clip`` writes, one per gradient and of its type; default: new tensors; pass ``grads`` to clip in place
    params   float32, one per gradient: what ``clip_adagrad`` updates
    accums   float32: Adagrad's accumulators (the reference starts them at 0.1)
    copies   bfloat16 / float16 / float32: rewritten from the updated parameters; entries may be None

    The constructor lays the list out on the device and waits for that; it cannot be captured into a graph.  The tensors
    are held and their CURRENT values are read by every call.  The calls enqueue on torch's current stream, allocate
    nothing once ``out`` is there, never synchronise, and may be captured.  Calls on one object (and replays of graphs that
    captured them) must be ordered one after the other: they share its partial sums.  The object may be dropped while eager
    calls are in flight, on any stream; it has to outlive the graphs that captured its calls, which read its table.

    A list may write a DNN scorer's own parameters, eagerly or in replayed graphs: from its construction on the scorer's
    fused step forms its transposed weight copies anew every time (other scorers keep theirs).  Such a list has to be built
    before a training step of that scorer is captured; afterwards it is refused with a RuntimeError."""

    def __init__(self, grads, out=None, params=None, accums=None, copies=None):
        if not torch.cuda.is_available():
            raise _lib.UltrError('GradientTensors needs an MI355X (HIP) device: there is no CPU path')
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError('GradientTensors lays its list out on the device: build it before the capture')
        self.grads = list(grads)
        self._index = torch.cuda.current_device()
        self.device = torch.device('cuda', self._index)
        self.params, self.accums, self.copies = (None if v is None else list(v) for v in (params, accums, copies))
        self.out = None if out is None else list(out)
        for k, g in enumerate(self.grads):
            if g.dtype not in _DTYPE or g.get_device() != self._index or not g.is_contiguous():
                raise ValueError('grads[%d]: a contiguous float32, bfloat16 or float16 tensor on %s expected, got %s on %s'
                                 % (k, self.device, g.dtype, g.device))
        for name, want in (('out', None), ('params', torch.float32), ('accums', torch.float32), ('copies', False)):
            self._check_role(name, want)
        self.norm = torch.zeros(1, dtype=torch.float32, device=self.device)
        self._norm_ptr = self.norm.data_ptr()
        self._tables = []
        self._build()

    def _check_role(self, name, dtype):
        tensors = getattr(self, name)
        if tensors is None:
            return
        if len(tensors) != len(self.grads):
            raise ValueError('%s: %d tensors for %d gradients' % (name, len(tensors), len(self.grads)))
        for k, (t, g) in enumerate(zip(tensors, self.grads)):
            if t is None and dtype is False:
                continue
            ok = t.dtype in _DTYPE if dtype is False else t.dtype == (g.dtype if dtype is None else dtype)
            if not ok or t.shape != g.shape or t.get_device() != self._index or not t.is_contiguous():
                raise ValueError('%s[%d]: contiguous %s %s on %s expected, got %s %s on %s'
                                 % (name, k, dtype or g.dtype, tuple(g.shape), self.device, t.dtype, tuple(t.shape), t.device))

    def _build(self):
        n = len(self.grads)
        rec = np.zeros(n, dtype=_REC)
        rec['grad'] = [g.data_ptr() for g in self.grads]
        rec['n'] = [g.numel() for g in self.grads]
        rec['grad_dtype'] = [_DTYPE[g.dtype] for g in self.grads]
        for name, tensors in (('out', self.out), ('param', self.params), ('accum', self.accums)):
            if tensors is not None:
                rec[name] = [t.data_ptr() for t in tensors]
        if self.copies is not None:
            rec['copy'] = [0 if t is None else t.data_ptr() for t in self.copies]
            rec['copy_dtype'] = [0 if t is None else _DTYPE[t.dtype] for t in self.copies]
        lib = _lib.lib()
        ptr = rec.ctypes.data_as(ctypes.POINTER(_lib.UltrTensor))
        nbytes = lib.ultr_tensors_table_bytes(ptr, n)
        if nbytes < 0:
            raise _lib.UltrError(lib.ultr_last_error().decode())
        table = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        plan = _lib.UltrTensorPlan()
        _lib.check(lib.ultr_tensors_plan(ptr, n, _lib.ptr(table), nbytes, plan, _lib.current_stream()), 'ultr_tensors_plan')
        self._tell_scorers(rec)
        # whichever stream uses the plan later finds it written
        torch.cuda.current_stream().synchronize()
        self._plan = ctypes.pointer(plan)
        self._tables.append(table)  # an earlier one stays: a captured graph may read it
        self._streams = set()  # that have used it

    @staticmethod
    def _tell_scorers(rec):
        """The scorers learn which memory the calls on this list write."""
        def memory():
            size = np.array([4, 2, 2], dtype=np.uint64)  # bytes of a DTYPE_*
            begin, end = [], []
            for name, each in (('out', size[rec['grad_dtype']]), ('param', 4), ('accum', 4), ('copy', size[rec['copy_dtype']])):
                there = (rec[name] != 0) & (rec['n'] > 0)
                begin.append(rec[name][there])
                end.append((rec[name] + rec['n'].astype(np.uint64) * np.asarray(each, dtype=np.uint64))[there])
            return np.concatenate(begin), np.concatenate(end)
        parameters_written(memory)

    def _stream(self):
        if _current_device() != self._index:
            raise ValueError('these tensors live on %s, the current device is cuda:%d' % (self.device, torch.cuda.current_device()))
        s = _lib.stream_of(self._index)
        if s not in self._streams:
            # dropped with calls in flight on this stream, the list's memory waits for them
            self._streams.add(s)
            stream = torch.cuda.current_stream()
            self._tables[-1].record_stream(stream)
            self.norm.record_stream(stream)
        return s

    def _denom(self, denom):
        if denom is None:
            return None
        if denom.get_device() != self._index or denom.dtype != torch.float32 or denom.numel() < 1:
            raise ValueError('denom: a float32 device scalar expected')
        return denom.data_ptr()

    def global_norm(self, denom=None, scale=1.0):
        """sqrt of the sum over all gradients of (scale / denom * g)^2, a device tensor [1] that the next call overwrites."""
        rc = _lib._lib.ultr_global_norm(self._plan, self._denom(denom), scale, self._norm_ptr, self._stream())
        if rc:
            _lib.check(rc, 'ultr_global_norm')
        return self.norm

    def clip(self, clip_norm, denom=None, scale=1.0):
        """-> (out, norm): out = scale / denom * g * clip_norm / max(norm, clip_norm).  A norm that
        is not finite makes every output NaN; clip_norm <= 0 does not clip."""
        if self.out is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError('clip: give ``out`` to the constructor before capturing')
            self._stream()  # the list is laid out on its own device
            self.out = [torch.empty_like(g) for g in self.grads]
            try:
                self._build()
            except Exception:
                self.out = None
                raise
        rc = _lib._lib.ultr_clip_by_global_norm(self._plan, self._denom(denom), scale, clip_norm, self._norm_ptr, self._stream())
        if rc:
            _lib.check(rc, 'ultr_clip_by_global_norm')
        return self.out, self.norm

    def clip_adagrad(self, clip_norm, learning_rate, denom=None, scale=1.0, l2=0.0, grad_strategy='ada'):
        """Clip and update the parameters in place (and the accumulators, and the copies); the gradients stay as they are.
        e = scale / denom * g + l2 * param; the norm is over e.  grad_strategy: 'ada' or 'sgd', as the hparam.
        -> norm, a device tensor [1] that the next call overwrites."""
        if self.params is None:
            raise ValueError('clip_adagrad: the list was built without params')
        strategy = _STRATEGY.get(grad_strategy)
        if strategy is None:
            raise ValueError("grad_strategy '%s' unknown (ada, sgd)" % grad_strategy)
        rc = _lib._lib.ultr_clip_adagrad_tensors(self._plan, self._denom(denom), scale, l2, clip_norm, learning_rate, strategy,
                                                 self._norm_ptr, self._stream())
        if rc:
            _lib.check(rc, 'ultr_clip_adagrad_tensors')
        return self.norm
