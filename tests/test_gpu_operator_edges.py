"""GPU tests (-m gpu) of calls at the edges of what the stand-alone layer norm and the tensor lists allow: memory that serves
two roles, values far from zero, sizes on both sides of where a pass changes.  Tolerances as in the two files whose reference
implementations these use."""
import pytest
import torch

from tests.test_gpu_tensor_list import BF16, F32, U, half_step, ref_norm, tensors, within

pytestmark = pytest.mark.gpu

MANY = [4096 * 2100 + 9, 5, 1, 70001]  # more chunks than a pass has workgroups


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_the_norm_as_the_denominator(dtype):
    """norm is both what the call divides by and where it writes: all of the list is divided by the old value."""
    from ultra_amd.learning_algorithm import GradientTensors
    grads = tensors(MANY, (dtype,), 1)
    plan = GradientTensors(grads, out=[torch.empty_like(g) for g in grads])
    apart = GradientTensors(grads, out=[torch.empty_like(g) for g in grads])
    for clip in (0.25, 2.0):
        old = plan.global_norm().clone()
        want, norm = apart.clip(clip, denom=old)
        got, same = plan.clip(clip, denom=plan.norm)
        assert torch.equal(norm, same) and abs(float(norm) - 1.0) <= 16 * U
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for o, g in zip(got, grads):
            w = g.double() / ref_norm(grads) * min(1.0, clip)
            within(o, w, 12 * U * w.abs() + half_step(dtype, w), 'out')  # norm 4 u, twice, and the clip's own 4 u


def test_a_denominator_that_the_call_overwrites():
    from ultra_amd import _lib
    from ultra_amd.learning_algorithm import GradientTensors
    for where in ('grad', 'param', 'accum', 'copy', 'param without a norm'):
        def make():
            grads, params = tensors(MANY, (F32,), 1), tensors(MANY, (F32,), 2)
            accums, copies = [t.abs().add_(0.1) for t in tensors(MANY, (F32,), 3)], [torch.zeros_like(p) for p in params]
            for role in (grads, params, accums, copies):
                role[2].fill_(8.0)
            return {'grad': grads, 'param': params, 'accum': accums, 'copy': copies}
        got, want = make(), make()
        one = torch.full((1,), 8.0, device='cuda')
        for lists, denom in ((got, got[where.split()[0]][2]), (want, one)):
            if where == 'grad':
                GradientTensors(lists['grad'], out=lists['grad']).clip(0.5, denom=denom)
                continue
            plan = GradientTensors(lists['grad'], params=lists['param'], accums=lists['accum'], copies=lists['copy'])
            if where == 'param without a norm':
                assert _lib.lib().ultr_clip_adagrad_tensors(plan._plan, denom.data_ptr(), 1.0, 0.01, 0.0, 0.05, _lib.OPT_ADAGRAD,
                                                            None, _lib.current_stream()) == 0
            else:
                plan.clip_adagrad(0.5, 0.05, denom=denom)
        torch.cuda.synchronize()
        assert float(one) == 8.0
        for role in got:
            assert all(torch.equal(a, b) for a, b in zip(got[role], want[role])), (where, role)


def scorers(count):
    """Equal small DNN scorers under DLA, one batch, each stepped twice: their fused steps have run and may keep weight copies."""
    from tests.test_gpu_step import PBM, make, settings
    from tests.util import SyntheticData
    data = SyntheticData(300, 10, 24, seed=11)
    exp = settings('DLA', '', 'hidden_layer_sizes=[64, 32]', Lmax=10, cutoff=10, feed_hparams='click_model_json=%s' % PBM)
    made = [make('DLA', data, exp, 64) for _ in range(count)]
    batch, _ = made[0][1].get_batch(data, check_validation=True)
    models = [m for m, _ in made]
    for m in models:
        assert m.model.fused_supported(64, 10)
        for _ in range(2):
            m.step(None, batch, False)
    return models, batch, [f for _, f in made]


def list_over(model):
    from ultra_amd.learning_algorithm import GradientTensors
    p = model.model.params
    half = p.numel() // 2
    gen = torch.Generator(device='cuda').manual_seed(5)
    grads = [torch.randn(n, generator=gen, device='cuda') for n in (half, p.numel() - half)]
    return GradientTensors(grads, params=[p[:half], p[half:]])


def test_a_replayed_update_of_a_scorers_parameters():
    """The graph writes the parameters, nothing else tells the scorer.  m2 takes the values through a copy that torch counts."""
    (m1, m2), batch, _feeds = scorers(2)
    plan = list_over(m1)
    plan.clip_adagrad(0.0, 0.5, grad_strategy='sgd')
    m2.model.params.copy_(m1.model.params)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan.clip_adagrad(0.0, 0.5, grad_strategy='sgd')
    for m in (m1, m2):
        m.step(None, batch, False)
    for _ in range(3):
        graph.replay()
        m2.model.params.copy_(m1.model.params)
        for m in (m1, m2):
            m.step(None, batch, False)
        assert torch.equal(m1.model.params, m2.model.params)


def test_an_update_between_replays_of_a_scorers_step():
    (m1, m2), batch, _feeds = scorers(2)
    plan = list_over(m1)
    for m in (m1, m2):
        m.enable_graph_replay(True)
        m.step(None, batch, False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m1.step(None, batch, False)
    for _ in range(3):
        plan.clip_adagrad(0.0, 0.5, grad_strategy='sgd')
        m2.model.params.copy_(m1.model.params)
        graph.replay()
        m2.step(None, batch, False)
        torch.cuda.synchronize()
        assert torch.equal(m1.model.params, m2.model.params)


def test_a_list_over_the_parameters_of_a_captured_step():
    (m1, m2), batch, _feeds = scorers(2)
    m1.enable_graph_replay(True)
    m1.step(None, batch, False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m1.step(None, batch, False)
    with pytest.raises(RuntimeError, match='before capturing'):
        list_over(m1)
    list_over(m2)  # of which no step was captured
    assert m1.model._wt_kept and not m2.model._wt_kept
