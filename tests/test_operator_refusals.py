"""What the stand-alone layer norm and tensor-list calls refuse, through the C ABI.  Arguments are checked on the host
before anything is launched, so this needs no GPU: the addresses below are never touched."""
import ctypes

import pytest

from ultra_amd import _lib

P = 1 << 20  # an aligned address that nothing dereferences
F32, BF16, F16 = _lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_F16


def last():
    return _lib.lib().ultr_last_error().decode()


def forward(**kw):
    a = dict(x=P, ldx=8, gamma=None, beta=None, M=2, N=8, eps=1e-3, xd=F32, wd=F32, y=2 * P, ldy=8, stats=None)
    a.update(kw)
    return _lib.lib().ultr_layer_norm_forward(a['x'], a['ldx'], a['gamma'], a['beta'], a['M'], a['N'], a['eps'], a['xd'], a['wd'],
                                              a['y'], a['ldy'], a['stats'], None)


@pytest.mark.parametrize('kw,rc,text', [
    (dict(x=None), -1, 'null x'), (dict(y=None), -1, 'null y'), (dict(M=-1), -1, 'M=-1'), (dict(N=0), -1, 'N=0'),
    (dict(N=65537, ldx=1 << 17, ldy=1 << 17), -2, 'too large'), (dict(ldx=7), -1, 'apart'), (dict(ldy=7), -1, 'apart'),
    (dict(ldx=0), -1, 'apart'), (dict(ldx=-8), -1, 'apart'), (dict(xd=3), -1, 'x_dtype'), (dict(wd=BF16), -1, 'w_dtype'),
    (dict(xd=BF16, wd=F16), -1, 'w_dtype'), (dict(eps=0.0), -1, 'eps'), (dict(eps=float('nan')), -1, 'eps'),
    (dict(x=P + 2), -1, 'aligned'), (dict(xd=F16, y=2 * P + 1), -1, 'aligned'), (dict(gamma=P + 1), -1, 'aligned'),
    (dict(stats=P + 4), -1, 'aligned'), (dict(y=P, ldy=9), -1, 'overlaps'), (dict(y=P + 32), -1, 'overlaps'),
])
def test_forward_refuses(kw, rc, text):
    assert forward(**kw) == rc
    assert text in last()


def test_no_rows_is_no_work():
    assert forward(M=0, x=None, y=None) == 0


def backward(**kw):
    a = dict(dy=P, lddy=8, x=2 * P, ldx=8, stats=3 * P, gamma=None, M=2, N=8, xd=F32, wd=F32, dx=4 * P, lddx=8, dg=5 * P, db=6 * P,
             ws=7 * P)
    a.update(kw)
    return _lib.lib().ultr_layer_norm_backward(a['dy'], a['lddy'], a['x'], a['ldx'], a['stats'], a['gamma'], a['M'], a['N'], a['xd'],
                                               a['wd'], a['dx'], a['lddx'], a['dg'], a['db'], a['ws'], None)


@pytest.mark.parametrize('kw,rc,text', [
    (dict(dy=None), -1, 'null dy'), (dict(x=None), -1, 'null x'), (dict(stats=None), -1, 'null stats'),
    (dict(dx=None, dg=None, db=None), -1, 'nothing'), (dict(M=100000, ws=None, dx=None), -1, 'workspace'), (dict(ws=P + 8), -1, 'aligned'),
    (dict(lddy=7), -1, 'apart'), (dict(lddx=7), -1, 'apart'), (dict(dx=P), -1, 'overlaps'), (dict(dx=2 * P), -1, 'overlaps'),
    (dict(dx=2 * P + 60), -1, 'overlaps'), (dict(stats=P + 4), -1, 'aligned'), (dict(xd=F16, wd=BF16), -1, 'w_dtype'),
    (dict(N=65537, ldx=1 << 17, lddy=1 << 17, lddx=1 << 17), -2, 'too large'), (dict(dg=5 * P + 2), -1, 'aligned'),
    (dict(db=5 * P + 28), -1, 'overlaps'), (dict(gamma=5 * P), -1, 'overlaps'), (dict(gamma=6 * P + 4), -1, 'overlaps'),
])
def test_backward_refuses(kw, rc, text):
    assert backward(**kw) == rc
    assert text in last()


def test_workspace_sizes():
    lib = _lib.lib()
    assert lib.ultr_layer_norm_workspace_bytes(-1, 8) == -1
    assert lib.ultr_layer_norm_workspace_bytes(8, 0) == -1
    for m in (0, 1, 7, 4096, 1 << 30):
        for n in (1, 136, 65536):
            assert lib.ultr_layer_norm_workspace_bytes(m, n) >= 0


def tensor(grad=P, out=None, param=None, accum=None, copy=None, n=16, gd=F32, cd=F32):
    return _lib.UltrTensor(grad, out, param, accum, copy, n, gd, cd)


def plan(*tensors, table=1 << 40, nbytes=1 << 20):
    arr = (_lib.UltrTensor * max(1, len(tensors)))(*tensors)
    return _lib.lib().ultr_tensors_plan(arr, len(tensors), table, nbytes, _lib.UltrTensorPlan(), None)


@pytest.mark.parametrize('t,text', [
    (tensor(n=-1), 'n=-1'), (tensor(grad=None), 'no gradient'), (tensor(gd=7), 'grad_dtype'), (tensor(grad=P + 2), 'aligned'),
    (tensor(out=2 * P + 1, gd=F16), 'aligned'), (tensor(param=2 * P + 2), 'aligned'), (tensor(copy=2 * P), 'copy'),
    (tensor(param=2 * P, copy=3 * P, cd=5), 'copy'), (tensor(out=P + 4), 'overlaps'), (tensor(param=P), 'overlaps'),
    (tensor(param=2 * P, accum=2 * P + 60), 'overlaps'), (tensor(param=2 * P, copy=2 * P), 'overlaps'),
])
def test_plan_refuses_a_tensor(t, text):
    assert plan(t) == -1
    assert text in last()


def test_plan_refuses_tensors_that_share_written_memory():
    # the same tensor twice: two workgroups would update it
    assert plan(tensor(param=2 * P, accum=3 * P), tensor(grad=4 * P, param=2 * P, accum=5 * P)) == -1 and 'overlaps' in last()
    assert plan(tensor(out=P), tensor(out=P)) == -1 and 'overlaps' in last()
    # one tensor's output is another one's gradient
    assert plan(tensor(out=2 * P), tensor(grad=2 * P + 32, out=3 * P)) == -1 and 'overlaps' in last()
    assert plan(tensor(grad=2 * P + 32, out=3 * P), tensor(out=2 * P)) == -1 and 'overlaps' in last()


def test_plan_refuses_tables():
    assert plan(tensor(), table=None) == -1
    assert plan(tensor(), table=(1 << 40) + 8) == -1 and 'aligned' in last()
    assert plan(tensor(), nbytes=64) == -1 and 'needed' in last()
    lib = _lib.lib()
    assert lib.ultr_tensors_table_bytes(None, 1) == -1
    assert lib.ultr_tensors_table_bytes(None, -1) == -1
    assert lib.ultr_tensors_table_bytes(None, 0) > 0
    assert lib.ultr_tensors_table_bytes(ctypes.byref(tensor(n=1 << 41)), 1) == -1


def test_calls_refuse_what_the_list_lacks():
    lib = _lib.lib()
    p = _lib.UltrTensorPlan(1 << 40, 1, 1, 0)
    assert lib.ultr_global_norm(None, None, 1.0, P, None) == -1
    assert lib.ultr_global_norm(p, None, 1.0, None, None) == -1
    assert lib.ultr_clip_by_global_norm(p, None, 1.0, 1.0, P, None) == -1 and 'lacks out' in last()
    assert lib.ultr_clip_by_global_norm(p, None, 1.0, float('nan'), P, None) == -1 and 'not a number' in last()
    assert lib.ultr_clip_adagrad_tensors(p, None, 1.0, 0.0, 1.0, 0.1, _lib.OPT_ADAGRAD, P, None) == -1 and 'lacks param accum' in last()
    p.has = 2
    assert lib.ultr_clip_adagrad_tensors(p, None, 1.0, 0.0, 1.0, 0.1, _lib.OPT_ADAGRAD, P, None) == -1 and 'lacks accum' in last()
    assert lib.ultr_clip_adagrad_tensors(p, None, 1.0, 0.0, 1.0, 0.1, 9, P, None) == -1 and 'grad_strategy' in last()


def test_the_python_record_is_the_abi_record():
    from ultra_amd.learning_algorithm.gradient_tensors import _REC
    assert _REC.itemsize == ctypes.sizeof(_lib.UltrTensor)
    for name, _ in _lib.UltrTensor._fields_:
        assert _REC.fields[name][1] == getattr(_lib.UltrTensor, name).offset
        assert _REC.fields[name][0].itemsize == getattr(_lib.UltrTensor, name).size


def test_a_scorer_refuses_half_precision_storage():
    from ultra_amd.ranking_model import DNN
    with pytest.raises(ValueError, match='compute_dtype'):
        DNN('compute_dtype=f16').create_variables(8, 'cpu')
