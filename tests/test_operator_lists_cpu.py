"""What a tensor list tells the scorers whose parameters it writes; no GPU needed."""
import numpy as np
import pytest


def scorer():
    from ultra_amd.ranking_model import DNN
    m = DNN('hidden_layer_sizes=[8]')
    m.create_variables(8, 'cpu')
    return m


def written(**roles):
    """A list of one tensor of four elements per role."""
    from ultra_amd.learning_algorithm.gradient_tensors import GradientTensors, _REC
    rec = np.zeros(2, dtype=_REC)  # the second one has no elements
    rec['n'] = [4, 0]
    for name, (address, dtype) in roles.items():
        rec[name][:] = address
        if name in ('out', 'copy'):
            rec['grad_dtype' if name == 'out' else 'copy_dtype'] = dtype
    GradientTensors._tell_scorers(rec)


@pytest.mark.parametrize('role,dtype,size', [('out', 0, 16), ('out', 1, 8), ('param', 0, 16), ('accum', 0, 16), ('copy', 0, 16), ('copy', 2, 8)])
def test_only_the_scorer_whose_parameters_are_written_stops_keeping_copies(role, dtype, size):
    near, other = scorer(), scorer()
    begin, end = near.params.data_ptr(), near.params.data_ptr() + 4 * near.params.numel()
    written(**{role: (begin - size, dtype)})
    written(**{role: (end, dtype)})
    assert near._wt_kept and other._wt_kept
    written(**{role: ((begin - size + 2) if role != 'copy' else end - 2, dtype)})
    assert not near._wt_kept and other._wt_kept
    written(**{role: (begin, dtype)})  # once more is no error


def test_gradients_are_not_written():
    m = scorer()
    written(grad=(m.params.data_ptr(), 0))
    assert m._wt_kept


def test_a_list_after_the_capture_is_refused():
    m, other = scorer(), scorer()
    m._wt_captured = other._wt_captured = True
    with pytest.raises(RuntimeError, match='before capturing'):
        written(param=(m.params.data_ptr() + 4, 0))
    first = scorer()
    written(param=(first.params.data_ptr() + 4, 0))  # before the capture: nothing that a graph could rely on
    first._wt_captured = True
    written(param=(first.params.data_ptr() + 4, 0))


def test_a_copied_scorer_is_known_too():
    import copy
    m = scorer()
    twin, alias = copy.deepcopy(m), copy.copy(m)
    written(param=(twin.params.data_ptr(), 0))
    assert not twin._wt_kept and m._wt_kept and alias._wt_kept
    written(param=(m.params.data_ptr(), 0))
    assert not m._wt_kept and not alias._wt_kept
