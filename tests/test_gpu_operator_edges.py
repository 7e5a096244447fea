"""GPU tests (-m gpu) of calls at the edges of what the stand-alone layer norm and the tensor lists allow: memory that serves
two roles, values far from zero, sizes on both sides of where a pass changes.  Tolerances as in the two files whose reference
implementations these use."""
import pytest
import torch

from tests.test_gpu_tensor_list import BF16, F16, F32, U, half_step, ref_norm, tensors, within

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


def ref_norm_rows(x, gamma, beta, eps=1e-3):
    """y and stats in 64 bits with their tolerances where rows lie far from zero.  D: additions in a row (16 entries a thread, more
    beyond 8192, then 6 in a wave and 4 between waves).  e_m: what is left of the mean's error.
    fp32: the first sum is off by delta = (D + 2) u max|x|, the deviations from it sum to its correction, (D + 4) u of their mean
    size, which is at most s + delta.
    16 bit: P entries are added in fp32, all of a row up to 2048 (bf16 8192), a wave's share beyond.  If the smallest that is not 0
    is at least A P / 2^13 (bf16 2^16), A the largest, all of them and their sums are multiples of one step (11 or 8 bits each)
    below 2^24 steps: exact.  Else two of them are at least A / 2 apart (P <= 4096), the squared deviations of these P are at
    least A^2 / 8, and their sum is off by at most D u P A; over N / P of them, by Cauchy, that is D u sqrt(8 P) s of the mean.
    Its quotient leaves as two floats: 4 u^2 of it.
    The variance: D + 6 roundings of sums of positive terms s^2 + delta^2, and what e_m changes."""
    xd = x.double()
    n = x.shape[-1]
    g = torch.ones(n, dtype=torch.float64, device='cuda') if gamma is None else gamma.double()
    b = torch.zeros(n, dtype=torch.float64, device='cuda') if beta is None else beta.double()
    first = xd[:, :1]
    mean = first + (xd - first).mean(-1, keepdim=True)  # exact for constant rows
    d = xd - mean
    var = d.square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    s, most = var.sqrt(), xd.abs().amax(-1, keepdim=True)
    dd = max(16, n / 1024) + 10
    if x.dtype == F32:
        delta = (dd + 2) * U * most
        e_m = (dd + 4) * U * (s + delta)
    else:
        delta = U * most
        p = n if n <= (8192 if x.dtype == BF16 else 2048) else 1024 if n <= 8192 else n / 16
        e_m = dd * U * (8 * p) ** 0.5 * s + 4 * U * U * most
    e_d = e_m + 2 * U * (d.abs() + delta)
    rel = ((dd + 6) * U * (var + delta ** 2) + 2 * (s + delta) * e_m + e_m ** 2) / (var + eps)
    tol_r = rel / 2 + rel ** 2 + 4 * U  # of rstd, relative, while rel < 1
    y = d * rstd * g + b
    tol = half_step(x.dtype, y) + g.abs() * rstd * (e_d * (1 + tol_r) + d.abs() * (tol_r + 4 * U)) + U * (y.abs() + (d * rstd * g).abs())
    return y, torch.cat([mean, rstd], -1), tol, torch.cat([e_m + U * mean.abs(), rstd * tol_r], -1)


@pytest.mark.parametrize('m', [9, 2051])  # from 2048 rows on a thread group works on two of them
@pytest.mark.parametrize('n', [1, 3, 5, 136, 700, 1023, 2048, 5003, 12345, 40001])
def test_rows_that_hardly_vary_far_from_zero(m, n):
    """Constant rows, rows of neighbouring values, rows with one entry far out; features before any scaling reach such values."""
    from ultra_amd.ranking_model import layer_norm
    from tests.test_gpu_layer_norm import weights
    if m > 1000 and n > 6000:
        m = 2049
    for t, values in ((F32, (123456.7, -1e6, 1e7, 16777217.0, 3e38, 0.1)), (BF16, (1e6, -3e38, 1e-3)), (F16, (65504.0, -777.0))):
        gen = torch.Generator(device='cuda').manual_seed(n)
        x = torch.empty((m, n), dtype=t, device='cuda')
        for k in range(m):
            if k >= 27:
                break
            v = values[k % len(values)]
            x[k] = v
            near = (k // len(values)) % 3
            if near and abs(v) < 1e18 and abs(v) < 65504:
                step = torch.finfo(t).eps * abs(v)
                if near == 1:  # up to three steps of the type above it
                    x[k] += (torch.randint(0, 4, (n,), generator=gen, device='cuda') * step).to(t)
                else:
                    x[k] = torch.randn(n, generator=gen, device='cuda').to(t)
                    x[k, n // 2] = v
        for k in range(27, m, 27):
            x[k:k + 27] = x[:min(27, m - k)]
        gamma, beta = weights(n, F32 if t == F32 else t, 1)
        y, stats = layer_norm(x, gamma, beta)
        ry, rs, ty, ts = ref_norm_rows(x, gamma, beta)
        within(stats, rs, ts, 'stats %s' % t)
        within(y, ry, ty, 'y %s' % t)
        assert torch.isfinite(y).all()  # at 3e38 too, where the sum of a row leaves fp32


def test_a_list_dropped_while_another_stream_uses_it():
    from ultra_amd.learning_algorithm import GradientTensors
    grads = tensors([4096 * 40 + 3, 5], (F32,), 1)
    want = ref_norm(grads)
    plan = GradientTensors(grads)
    table, nbytes, norm = plan._tables[-1].data_ptr(), plan._tables[-1].numel(), plan.norm
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200 * 1000 * 1000)  # about 0.1 s
        plan.global_norm()
    done = side.record_event()
    del plan
    others = [torch.full((nbytes,), 255, dtype=torch.uint8, device='cuda') for _ in range(8)]
    if not done.query():
        assert all(t.data_ptr() != table for t in others)
    torch.cuda.synchronize()
    assert abs(float(norm) - want) <= 4 * U * want


@pytest.mark.parametrize('t', [F32, BF16])
@pytest.mark.parametrize('m,n', [(7, 5), (3000, 136), (40, 1030), (1100, 8201)])
def test_columns_of_one_table(t, m, n):
    """x, the output and the gradients side by side in one table: no rows overlap."""
    from tests.test_gpu_layer_norm import ref_backward, ref_forward, weights
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    gen = torch.Generator(device='cuda').manual_seed(1)
    table = torch.randn((m, 4 * n + 3), generator=gen, device='cuda').to(t)
    x, dy, y, dx = (table[:, a:a + n] for a in (1, n + 1, 2 * n + 2, 3 * n + 2))
    gamma, beta = weights(n, F32, 2)
    before = table.clone()
    got, stats = layer_norm(x, gamma, beta, out=y)
    ry, _, ty, _ = ref_forward(before[:, 1:1 + n], gamma, beta)
    within(got, ry, ty, 'y')
    _, dg, db = layer_norm_backward(dy, x, stats, gamma, d_x=dx)
    rx, rg, rb, tx, tg, tb = ref_backward(before[:, n + 1:2 * n + 1], before[:, 1:1 + n], stats, gamma)
    within(dx, rx, tx, 'dx')
    within(dg, rg, tg + half_step(F32, rg), 'd_gamma')
    within(db, rb, tb + half_step(F32, rb), 'd_beta')
    for a, b in ((0, 2 * n + 1), (2 * n + 1, 2 * n + 2), (4 * n + 2, 4 * n + 3)):
        assert torch.equal(table[:, a:b], before[:, a:b])
    # in the other order, and the workspace behind a matrix that ends before it
    z = table[:, 0:n]
    layer_norm(y, out=z)
    with pytest.raises(Exception, match='overlaps'):
        layer_norm(x, out=table[:, 2:2 + n])


def test_python_calls_that_share_memory():
    from ultra_amd import _lib
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    x, dy = torch.randn((6, 8), device='cuda'), torch.randn((6, 8), device='cuda')
    _, stats = layer_norm(x)
    for call in (lambda: layer_norm(x, gamma=x[0], out=x), lambda: layer_norm(x, stats=x.view(-1)[:12].view(6, 2)),
                 lambda: layer_norm_backward(dy, x, stats, d_gamma=dy[1]), lambda: layer_norm_backward(dy, x, stats, gamma=x[2], d_x=x),
                 lambda: layer_norm_backward(dy, x, stats, d_beta=stats.view(-1)[:8])):
        with pytest.raises(_lib.UltrError, match='overlaps'):
            call()


def test_what_a_list_moves_is_counted_in_bytes():
    from ultra_amd.learning_algorithm import GradientTensors
    tiny = GradientTensors(list(torch.randn(200000, device='cuda').split(10)))
    out, norm = tiny.clip(1.0)
    p = tiny._plan.contents
    assert (p.n_chunks, p.clip_bytes, p.update_bytes, p.keep_from) == (20000, 200000 * 8, 200000 * 12, 0)
    want = ref_norm(tiny.grads)
    assert abs(float(norm) - want) <= 4 * U * want
    within(torch.cat(out), torch.cat(tiny.grads).double() / want, 4 * U * torch.cat(tiny.grads).abs().double() + half_step(F32, norm), 'out')
    mixed = [torch.zeros(n, dtype=t, device='cuda') for n, t in ((4097, BF16), (1000, F32), (0, F16))]
    plan = GradientTensors(mixed, params=[torch.zeros(m.shape, device='cuda') for m in mixed],
                           accums=[torch.zeros(m.shape, device='cuda') for m in mixed],
                           copies=[torch.zeros(4097, dtype=F16, device='cuda'), None, None])._plan.contents
    assert (plan.n_chunks, plan.clip_bytes, plan.update_bytes, plan.keep_from) == (3, 4097 * 4 + 1000 * 8, 4097 * 20 + 1000 * 20, 0)


@pytest.mark.parametrize('sizes,dtypes,chunks', [
    ([150000001, 4097], (BF16,), 36622 + 2 - 32768 + 1), ([70000003, 9], (F32,), 17090 + 1 - 16384 + 1),
    ([40000001, 70000000, 8193], (F32, BF16), None), ([5, 300000001], (F16,), 1 + 73243 - 32768)])
def test_first_passes_that_change_over(sizes, dtypes, chunks):
    """Gradients beyond 256 MB: the first ones are read past the caches, the last 256 MB are not.  Every chunk is counted once,
    with the parameters' part of the norm too."""
    from ultra_amd.learning_algorithm import GradientTensors
    grads, params = tensors(sizes, dtypes, 1, aligned=False), tensors(sizes, (F32,), 2, aligned=False)
    plan = GradientTensors(grads, out=[torch.empty_like(g) for g in grads], params=params)
    p = plan._plan.contents
    assert 0 < p.keep_from < p.n_chunks
    if chunks is not None:
        assert abs(p.keep_from - chunks) <= 1
    kept = sum(g.numel() * g.element_size() for g in grads)
    assert kept > 256 << 20 and p.clip_bytes == 2 * kept
    want = ref_norm(grads)
    out, norm = plan.clip(1.0)
    assert abs(float(norm) - want) <= 4 * U * want and abs(float(plan.global_norm()) - want) <= 4 * U * want
    for o, g in zip(out, grads):
        w = g.double() / want
        within(o, w, 4 * U * w.abs() + half_step(g.dtype, w), 'out')
        del w
    with_l2 = sum(float((g.double() + 0.01 * q.double()).square().sum()) for g, q in zip(grads, params)) ** 0.5
    before = [q.clone() for q in params]
    got = plan.clip_adagrad(1.0, 0.5, l2=0.01, grad_strategy='sgd')
    assert abs(float(got) - with_l2) <= 8 * U * with_l2
    for q, b, g in zip(params, before, grads):
        step = (g.double() + 0.01 * b.double()) * (0.5 / with_l2)
        tol = 9 * U * (g.double().abs() + 0.01 * b.double().abs()) * (0.5 / with_l2) + U * 2 * b.abs()
        within(q, b.double() - step, tol, 'param')


def test_a_list_whose_outputs_could_not_be_laid_out(monkeypatch):
    from ultra_amd import _lib
    from ultra_amd.learning_algorithm import GradientTensors
    grads = tensors([5000, 3], (F32,), 1)
    want = ref_norm(grads)
    plan = GradientTensors(grads)

    def fails(rc, what):
        raise _lib.UltrError('no')
    with monkeypatch.context() as m:
        m.setattr(_lib, 'check', fails)
        with pytest.raises(_lib.UltrError):
            plan.clip(1.0)
    assert plan.out is None and len(plan._tables) == 1
    assert abs(float(plan.global_norm()) - want) <= 4 * U * want
    out, _ = plan.clip(want / 2)
    within(out[0], grads[0].double() / 2, 5 * U * grads[0].double().abs(), 'out')


def test_a_first_clip_on_another_device(monkeypatch):
    """The outputs are laid out by kernels, on the list's device only."""
    from ultra_amd.learning_algorithm import GradientTensors, gradient_tensors
    plan = GradientTensors(tensors([5000, 3], (F32,), 1))
    with monkeypatch.context() as m:
        m.setattr(gradient_tensors, '_current_device', lambda: plan._index + 1)
        with pytest.raises(ValueError, match='current device'):
            plan.clip(1.0)
    assert plan.out is None and len(plan._tables) == 1
    plan.clip(1.0)


# ---- forms that other tests pass by ---------------------------------------------------------------------------------------
@pytest.mark.parametrize('m,n', [(2048, 300), (2049, 700), (3001, 1030), (2051, 2048), (2048, 4096), (2049, 4097), (2050, 5003), (2049, 8200),
                                 (2051, 16384), (2049, 16385), (2100, 1052)])
def test_forward_of_two_rows_a_thread_group(m, n):
    """From 2048 rows on a thread group forms two rows: whole waves, several waves, odd last rows, odd widths, in a table, in place."""
    from tests.test_gpu_layer_norm import TYPES, ref_forward, rows, weights
    from ultra_amd.ranking_model import layer_norm
    for k, (t, w) in enumerate(TYPES):
        x, _ = rows(m, n, t, k, gap=5 * (k % 2), shift=k % 3, scale=1.5, offset=0.7)
        gamma, beta = weights(n, w, k + 10)
        ry, rs, ty, ts = ref_forward(x, gamma, beta)
        y, buf = rows(m, n, t, 99, gap=3, shift=1)
        before = buf.clone()
        _, stats = layer_norm(x, gamma, beta, out=y)
        within(stats, rs, ts, 'stats %s' % t)
        within(y, ry, ty, 'y %s %s' % (t, w))
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:].view(m, n + 3)[:, :n] = False
        assert torch.equal(buf[keep], before[keep])
        layer_norm(x, gamma, beta, out=x)
        assert torch.equal(x, y)


@pytest.mark.parametrize('m,n', [(1025, 16392), (1100, 16385), (1030, 20000), (2049, 17001), (1025, 32768), (1026, 40007), (1025, 65536)])
def test_backward_of_many_wide_rows(m, n):
    """16-bit rows beyond 16384 and fp32 rows beyond 8192, more than 1024 of them: column tiles times row slices."""
    from tests.test_gpu_layer_norm import TYPES, ref_backward, ref_forward, rows, weights
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    for k, (t, w) in enumerate(TYPES):
        x, _ = rows(m, n, t, k, gap=3 * (k % 2), shift=k % 2, scale=1.5, offset=0.4)
        dy, _ = rows(m, n, t, k + 50)
        gamma, _ = weights(n, w, k)
        _, stats = layer_norm(x)
        _, rs, _, ts = ref_forward(x, None, None)
        within(stats, rs, ts, 'stats')
        d_x, buf = rows(m, n, t, 99, gap=5, shift=1)
        before = buf.clone()
        dx, dg, db = layer_norm_backward(dy, x, stats, gamma, d_x=d_x)
        rx, rg, rb, tx, tg, tb = ref_backward(dy, x, stats, gamma)
        within(dx, rx, tx, 'dx %s' % t)
        within(dg, rg, tg + half_step(w, rg), 'd_gamma %s' % w)
        within(db, rb, tb + half_step(w, rb), 'd_beta %s' % w)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:].view(m, n + 5)[:, :n] = False
        assert torch.equal(buf[keep], before[keep])
        del rx, tx, keep, before
        again = layer_norm_backward(dy, x, stats, gamma)
        assert all(torch.equal(p, q) for p, q in zip((dx, dg, db), again))
        only = layer_norm_backward(dy, x, stats, gamma, need=(False, True, True))
        assert torch.equal(only[1], dg) and torch.equal(only[2], db)
        only = layer_norm_backward(dy, x, stats, gamma, need=(True, False, False))
        assert torch.equal(only[0], dx)


@pytest.mark.parametrize('m,n', [(16, 136), (700, 512), (3000, 700), (1030, 8200), (600, 9001)])
def test_statistics_that_a_gradient_takes(m, n):
    """The gradient's tests take the forward pass's statistics as given; here they are checked at such sizes."""
    from tests.test_gpu_layer_norm import TYPES, ref_forward, rows
    from ultra_amd.ranking_model import layer_norm
    for k, (t, _) in enumerate(TYPES):
        x, _ = rows(m, n, t, k, scale=1.5, offset=0.4)
        y, stats = layer_norm(x)
        ry, rs, ty, ts = ref_forward(x, None, None)
        within(stats, rs, ts, 'stats')
        within(y, ry, ty, 'y')
