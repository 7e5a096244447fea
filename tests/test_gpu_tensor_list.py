"""GPU tests (-m gpu) of the norm, the clip and the update over a list of tensors, against their formulas in 64 bits.

Tolerances: u = 2^-24.  e = scale * g has two roundings (the scale's and the product's), one more with the clip factor and one
for the factor itself: 4 u relative.  The norm sums squares of fp32 products in 64 bits: 2 u for the product and the scale, one
for the result, doubled: 4 u.  The update's step lr e / sqrt(a): e 4 u, a 9 u of which the root takes half, three operations:
12 u.  A stored value adds half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(t, v):
    f = torch.finfo(t)
    return f.eps / 2 * v.abs() + f.smallest_normal * f.eps / 2


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    if bad.any():
        k = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError('%s: %d of %d off, first at %d: got %r want %r tol %r' % (
            what, int(bad.sum()), bad.numel(), k, got.reshape(-1)[k].item(), want.reshape(-1)[k].item(), tol.reshape(-1)[k].item()))


def tensors(sizes, dtypes, seed, scale=1.0, aligned=True):
    g = torch.Generator(device='cuda').manual_seed(seed)
    out = []
    for k, n in enumerate(sizes):
        t = dtypes[k % len(dtypes)]
        v = torch.randn(n, generator=g, device='cuda') * scale * 10.0 ** -(k % 3)
        if aligned:
            out.append(v.to(t))
        else:  # anywhere the element type allows, with memory in front and behind
            buf = torch.empty(n + 7, dtype=t, device='cuda')
            out.append(buf[1 + k % 5:1 + k % 5 + n])
            out[-1].copy_(v)
    return out


def ref_norm(grads, scale=1.0):
    return sum(float((g.double() * scale).square().sum()) for g in grads) ** 0.5


SIZES = {
    'one': [1], 'empty': [], 'without elements': [0, 0], 'a few': [1, 0, 5, 3], 'one chunk': [4095, 4096, 4097, 8192, 8193],
    'small': [136 * 512, 512, 136, 136, 512 * 256, 256, 512, 512], 'many': [(k * 37) % 701 for k in range(1300)],
    'large': [3000001, 17, 1 << 20, 70000, 5], 'past the grid': [4096 * 2100 + 9, 1],
}


@pytest.mark.parametrize('name', sorted(SIZES))
@pytest.mark.parametrize('dtypes', [(F32,), (BF16,), (F16,), (F32, F16, BF16)])
def test_norm_and_clip(name, dtypes):
    from ultra_amd.learning_algorithm import GradientTensors
    for aligned in (True, False):
        grads = tensors(SIZES[name], dtypes, 3, aligned=aligned)
        kept = [g.clone() for g in grads]
        plan = GradientTensors(grads, out=tensors(SIZES[name], dtypes, 4, aligned=aligned))
        want = ref_norm(grads)
        assert abs(float(plan.global_norm()) - want) <= 4 * U * want
        denom = torch.full((1,), 3.0, device='cuda')
        assert abs(float(plan.global_norm(denom, 0.5)) - want / 6) <= 4 * U * want / 6
        for clip in (0.5 * want, 2.0 * want, 0.0):
            f = min(1.0, clip / want) if clip > 0 else 1.0
            out, norm = plan.clip(clip)
            assert abs(float(norm) - want) <= 4 * U * want
            for k, (o, g) in enumerate(zip(out, grads)):
                w = g.double() * f
                within(o, w, 4 * U * w.abs() + half_step(g.dtype, w), 'out %d at clip %g' % (k, clip))
                if f == 1.0:
                    assert torch.equal(o, g)
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))


def test_clip_in_place_and_new_tensors():
    from ultra_amd.learning_algorithm import GradientTensors
    sizes = SIZES['a few'] + SIZES['one chunk']
    grads = tensors(sizes, (F32, BF16, F16), 5, aligned=False)
    want, kept = ref_norm(grads), [g.clone() for g in grads]
    made, norm = GradientTensors(grads).clip(0.25 * want, scale=2.0)
    assert abs(float(norm) - 2 * want) <= 4 * U * 2 * want
    out, _ = GradientTensors(grads, out=grads).clip(0.25 * want, scale=2.0)
    assert all(a is b for a, b in zip(out, grads))
    assert all(torch.equal(a, b) for a, b in zip(grads, made))
    for o, g in zip(made, kept):
        within(o, g.double() * 0.25, 5 * U * g.double().abs() + half_step(g.dtype, g.double() * 0.25), 'out')


@pytest.mark.parametrize('value', [1e25, 1e-25, 3e38, 1e-40])
def test_norms_whose_squares_leave_fp32(value):
    from ultra_amd.learning_algorithm import GradientTensors
    grads = [torch.full((5000,), value, device='cuda'), torch.full((3,), -value, device='cuda')]
    want = ref_norm(grads)
    got = float(GradientTensors(grads).global_norm())
    assert got == float('inf') if want > 3.4e38 else abs(got - want) <= 4 * U * want + 2.0 ** -150
    if 1e-30 < want < 3e38:
        out, _ = GradientTensors(grads).clip(want / 2)
        within(out[0], grads[0].double() / 2, 5 * U * grads[0].double(), 'out')


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
def test_a_norm_that_is_not_finite(bad):
    from ultra_amd.learning_algorithm import GradientTensors
    grads = tensors([10, 5000, 3], (F32, BF16), 1)
    grads[1][4500] = bad
    plan = GradientTensors(grads)
    out, norm = plan.clip(1.0)
    assert not torch.isfinite(norm).any()
    assert all(torch.isnan(o).all() for o in out)
    out, _ = plan.clip(0.0)  # not clipped: the others keep their values
    assert torch.equal(out[0], grads[0]) and torch.equal(out[2], grads[2])
    # an element that the norm does not know of: a tensor without elements has no values
    assert float(GradientTensors([torch.empty(0, device='cuda'), torch.ones(4, device='cuda')]).global_norm()) == 2.0


def ref_update(grads, params, accums, scale, l2, clip, lr, ada):
    e = [g.double() * scale + l2 * p.double() for g, p in zip(grads, params)]
    et = [(g.double() * scale).abs() + (l2 * p.double()).abs() for g, p in zip(grads, params)]
    norm = sum(float(v.square().sum()) for v in e) ** 0.5
    f = min(1.0, clip / norm) if clip > 0 and norm > 0 else 1.0
    res = []
    for v, vt, p, a in zip(e, et, params, accums):
        v, vt = v * f, vt * f
        if ada:
            acc = a.double() + v.square()
            step = lr * v / acc.sqrt()
            tol_a = 2 * U * acc + 9 * U * vt * v.abs()
            tol = (4 * vt + 9 * v.abs()) * U * lr / acc.sqrt()
        else:
            acc, step, tol_a, tol = a.double(), lr * v, 0 * v, 7 * U * lr * vt
        new = p.double() - step
        res.append((new, tol + U * (new.abs() + p.double().abs()), acc, tol_a))
    return norm, res


@pytest.mark.parametrize('name', sorted(SIZES))
@pytest.mark.parametrize('l2', [0.0, 0.01])
@pytest.mark.parametrize('strategy', ['ada', 'sgd'])
def test_update(name, l2, strategy):
    from ultra_amd.learning_algorithm import GradientTensors
    for dtypes, clip, aligned in (((F32,), 0.7, True), ((BF16, F32, F16), 1e6, False), ((F16,), 0.0, True), ((BF16,), 0.3, False)):
        sizes = SIZES[name]
        grads, params = tensors(sizes, dtypes, 1, aligned=aligned), tensors(sizes, (F32,), 2, aligned=aligned)
        accums = [t.abs().add_(0.1) for t in tensors(sizes, (F32,), 3, aligned=True)]
        copies = [None if k % 3 == 2 else t for k, t in enumerate(tensors(sizes, (BF16, F16), 4, aligned=aligned))]
        kept = [g.clone() for g in grads]
        acc_before = [a.clone() for a in accums]
        norm, ref = ref_update(grads, params, accums, 2.0 / 64, l2, clip, 0.05, strategy == 'ada')
        plan = GradientTensors(grads, params=params, accums=accums if strategy == 'ada' else None, copies=copies)
        got = plan.clip_adagrad(clip, 0.05, denom=torch.full((1,), 64.0, device='cuda'), scale=2.0, l2=l2, grad_strategy=strategy)
        assert abs(float(got) - norm) <= 8 * U * norm
        for k, (p, a, c, (rp, tp, ra, ta)) in enumerate(zip(params, accums, copies, ref)):
            within(p, rp, tp, 'param %d' % k)
            within(a, ra, ta, 'accum %d' % k)
            if c is not None:
                assert torch.equal(c, p.to(c.dtype)), 'copy %d' % k
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
        if strategy == 'sgd':
            assert all(torch.equal(a, b) for a, b in zip(accums, acc_before))


def test_update_agrees_with_the_flat_call():
    """One tensor: the arithmetic of ultr_clip_adagrad, so nearly its bits; the norms' orders of summation differ."""
    from ultra_amd import _lib
    from ultra_amd.learning_algorithm import GradientTensors
    n = 70001
    g, p = tensors([n], (F32,), 1)[0], tensors([n], (F32,), 2)[0]
    a = torch.full((n,), 0.1, device='cuda')
    flat = [t.clone() for t in (p, a)]
    ws, norm = torch.zeros(2048, device='cuda'), torch.zeros(1, device='cuda')
    _lib.check(_lib.lib().ultr_clip_adagrad(_lib.ptr(flat[0]), _lib.ptr(flat[1]), _lib.ptr(g), n, None, 0.25, 0.0, 5.0, 0.05,
                                            _lib.OPT_ADAGRAD, _lib.ptr(norm), _lib.ptr(ws), _lib.current_stream()), 'flat')
    got = GradientTensors([g], params=[p], accums=[a]).clip_adagrad(5.0, 0.05, scale=0.25)
    assert abs(float(got) - float(norm)) < 1e-5 * float(norm)
    assert (p - flat[0]).abs().max() < 1e-6 and ((a - flat[1]).abs() <= 1e-5 * flat[1]).all()


def test_update_with_a_norm_that_is_not_finite():
    from ultra_amd.learning_algorithm import GradientTensors
    grads, params = tensors([4, 5000], (F32,), 1), tensors([4, 5000], (F32,), 2)
    accums = [torch.full_like(p, 0.1) for p in params]
    grads[0][1] = float('nan')
    GradientTensors(grads, params=params, accums=accums).clip_adagrad(1.0, 0.05)
    assert all(torch.isnan(p).all() for p in params)


def test_more_than_2_31_elements():
    from ultra_amd.learning_algorithm import GradientTensors
    n = (1 << 31) + 4101
    g = torch.zeros(n, dtype=BF16, device='cuda')
    at = torch.tensor([0, 4095, 4096, (1 << 31) - 1, 1 << 31, n - 1], device='cuda')
    g[at] = torch.tensor([1.0, 2.0, 2.0, 4.0, 4.0, 8.0], dtype=BF16, device='cuda')
    out, norm = GradientTensors([g, torch.ones(3, device='cuda')]).clip(1.0)
    want = (1 + 4 + 4 + 16 + 16 + 64 + 3.0) ** 0.5
    assert abs(float(norm) - want) < 1e-6 * want
    w = g[at].double() / want
    within(out[0][at], w, 4 * U * w + half_step(BF16, w), 'far elements')
    assert int((out[0] != 0).sum()) == 6


def test_captured_and_replayed():
    from ultra_amd.learning_algorithm import GradientTensors
    sizes = SIZES['small'] + [1, 0, 70001]
    grads, params = tensors(sizes, (F32, BF16), 1), tensors(sizes, (F32,), 2)
    accums = [torch.full_like(p, 0.1) for p in params]
    start = [t.clone() for t in params + accums]
    plan = GradientTensors(grads, out=[torch.empty_like(g) for g in grads], params=params, accums=accums)
    denom = torch.ones(1, device='cuda')

    def step():
        plan.clip(0.5, denom)
        return plan.clip_adagrad(0.5, 0.05, denom)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()

    def reset():
        for t, s in zip(params + accums, start):
            t.copy_(s)
    for k in range(4):
        for g, v in zip(grads, tensors(sizes, (F32,), 40 + k)):
            g.copy_(v)
        denom.fill_(1.0 + k)
        reset()
        graph.replay()
        got = [t.clone() for t in plan.out + params + accums + [plan.norm]]
        torch.cuda.synchronize()
        reset()
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, plan.out + params + accums + [plan.norm]))


def test_a_graph_outlives_the_list_it_was_captured_with():
    from ultra_amd.learning_algorithm import GradientTensors
    grads = tensors(SIZES['small'], (F32,), 1)
    plan = GradientTensors(grads)
    plan.global_norm()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.global_norm()
    plan.clip(1.0)  # makes the outputs and lays the list out again
    waste = [torch.full((1 << 16,), 255, dtype=torch.uint8, device='cuda') for _ in range(64)]
    for k in range(3):
        grads[0].mul_(2.0)
        plan.norm.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = ref_norm(grads)
        assert abs(float(plan.norm) - want) <= 4 * U * want
    del waste


def test_what_the_c_calls_leave_out():
    """No norm wanted, none formed, an empty list, scalars, a plan laid out by the C call itself."""
    import ctypes
    from ultra_amd import _lib
    from ultra_amd.learning_algorithm import GradientTensors
    lib, st = _lib.lib(), _lib.current_stream()
    grads, params = tensors([4099, 3], (F16, F32), 1), tensors([4099, 3], (F32,), 2)
    out = [torch.empty_like(g) for g in grads]
    rec = (_lib.UltrTensor * 2)(*[_lib.UltrTensor(g.data_ptr(), o.data_ptr(), p.data_ptr(), None, None, g.numel(), _lib.DTYPE_F16 if g.dtype == F16 else _lib.DTYPE_F32, 0)
                                  for g, o, p in zip(grads, out, params)])
    nbytes = lib.ultr_tensors_table_bytes(rec, 2)
    table = torch.full((nbytes,), 255, dtype=torch.uint8, device='cuda')
    plan = _lib.UltrTensorPlan()
    assert lib.ultr_tensors_plan(rec, 2, table.data_ptr(), nbytes, ctypes.byref(plan), st) == 0
    assert plan.has == 3 and plan.n_tensors == 2 and plan.n_chunks == 3
    ctypes.memset(rec, 255, ctypes.sizeof(rec))  # the list may be dropped at once
    want = ref_norm(grads)
    assert lib.ultr_clip_by_global_norm(ctypes.byref(plan), None, 1.0, want / 4, None, st) == 0
    for o, g in zip(out, grads):
        within(o, g.double() / 4, 4 * U * g.double().abs() + half_step(g.dtype, g.double() / 4), 'out')
    before = [p.double() for p in params]
    assert lib.ultr_clip_adagrad_tensors(ctypes.byref(plan), None, 1.0, 0.0, 0.0, 0.5, _lib.OPT_SGD, None, st) == 0  # one launch
    for p, b, g in zip(params, before, grads):
        within(p, b - 0.5 * g.double(), 4 * U * (b.abs() + g.double().abs()), 'param')
    assert lib.ultr_clip_adagrad_tensors(ctypes.byref(plan), None, 1.0, 0.0, 1.0, 0.5, _lib.OPT_ADAGRAD, None, st) == -1
    empty = GradientTensors([], out=[], params=[], accums=[])
    assert float(empty.global_norm()) == 0 and empty.clip(1.0)[0] == [] and float(empty.clip_adagrad(1.0, 0.1)) == 0
    scalar, vector = torch.tensor(3.0, device='cuda'), torch.tensor([4.0], device='cuda')
    got, norm = GradientTensors([scalar, vector]).clip(1.0)
    assert float(norm) == 5.0 and got[0].shape == () and abs(float(got[0]) - 0.6) <= 1e-7 and abs(float(got[1]) - 0.8) <= 1e-7


def test_a_scorers_own_parameters_in_a_list():
    """The fused step streams copies of the weights that its own update keeps current: an update through a list must not leave
    them stale.  The second model takes the same values through a copy that torch knows of."""
    from tests.test_gpu_step import PBM, make, settings
    from tests.util import SyntheticData
    from ultra_amd.learning_algorithm import GradientTensors
    data = SyntheticData(300, 10, 24, seed=11)
    exp = settings('DLA', '', 'hidden_layer_sizes=[64, 32]', Lmax=10, cutoff=10, feed_hparams='click_model_json=%s' % PBM)
    m1, feed = make('DLA', data, exp, 64)
    m2, _ = make('DLA', data, exp, 64)
    assert m1.model.fused_supported(64, 10)
    batch, _ = feed.get_batch(data, check_validation=True)
    for m in (m1, m2):
        m.step(None, batch, False)
    p = m1.model.params
    half = p.numel() // 2
    plan = GradientTensors([torch.randn(half, device='cuda'), torch.randn(p.numel() - half, device='cuda')], params=[p[:half], p[half:]])
    for _ in range(2):
        plan.clip_adagrad(0.0, 0.5, grad_strategy='sgd')
        m2.model.params.copy_(p)
        for m in (m1, m2):
            m.step(None, batch, False)
        assert torch.equal(m1.model.params, m2.model.params)


def test_two_lists_in_flight():
    from ultra_amd.learning_algorithm import GradientTensors
    lists = []
    for k in range(2):
        grads = tensors(SIZES['large'] + SIZES['many'][:300], (F32, BF16), k)
        plan = GradientTensors(grads, out=[torch.empty_like(g) for g in grads])
        plan.clip(1.0)
        lists.append((plan, [o.clone() for o in plan.out], plan.norm.clone()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lists]
    for _ in range(3):
        for s, (plan, _, _) in zip(streams, lists):
            with torch.cuda.stream(s):
                plan.clip(1.0)
    torch.cuda.synchronize()
    for plan, out, norm in lists:
        assert torch.equal(plan.norm, norm) and all(torch.equal(a, b) for a, b in zip(plan.out, out))


def test_python_refusals():
    from ultra_amd import _lib
    from ultra_amd.learning_algorithm import GradientTensors
    g, p = torch.randn(6, 4, device='cuda'), torch.randn(6, 4, device='cuda')
    for kw in (dict(grads=[g.cpu()]), dict(grads=[g.double()]), dict(grads=[g.t()]), dict(grads=[g], out=[]),
               dict(grads=[g], out=[p.half()]), dict(grads=[g], params=[p.half()]), dict(grads=[g], params=[p.view(4, 6)]),
               dict(grads=[g], params=[p], accums=[p.cpu()]), dict(grads=[g], params=[p], copies=[p.long()])):
        with pytest.raises(ValueError):
            GradientTensors(**kw)
    for kw in (dict(grads=[g, p], params=[p, p.clone()]), dict(grads=[g, g], out=[p, p]), dict(grads=[g], copies=[p])):
        with pytest.raises(_lib.UltrError):
            GradientTensors(**kw)
    with pytest.raises(ValueError):
        GradientTensors([g]).clip_adagrad(1.0, 0.1)
    with pytest.raises(_lib.UltrError):
        GradientTensors([g], params=[p]).clip_adagrad(1.0, 0.1)  # Adagrad without accumulators
    with pytest.raises(ValueError):
        GradientTensors([g], params=[p]).clip_adagrad(1.0, 0.1, grad_strategy='adam')
    with pytest.raises(ValueError):
        GradientTensors([g]).clip(1.0, denom=torch.ones(1))


def test_a_ranker_of_ones_own_trains():
    """Layer norm, a product, layer norm, scores; softmax loss over lists; backward; clip + Adagrad over the separate
    variables: a few steps together, each against the same step in 64 bits from the same state."""
    from ultra_amd.learning_algorithm import GradientTensors
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    B, L, F, H, lr, clip = 64, 10, 136, 96, 0.05, 0.5
    gen = torch.Generator(device='cuda').manual_seed(0)
    x = torch.rand((B * L, F), generator=gen, device='cuda') * 2 - 1
    clicks = (torch.rand((B, L), generator=gen, device='cuda') < 0.3).float()
    W, v = torch.randn((F, H), generator=gen, device='cuda') * F ** -0.5, torch.randn((H, 1), generator=gen, device='cuda') * H ** -0.5
    params = [torch.ones(F, device='cuda'), torch.zeros(F, device='cuda'), W, torch.ones(H, device='cuda'), torch.zeros(H, device='cuda'), v]
    grads = [torch.empty_like(p) for p in params]
    accums = [torch.full_like(p, 0.1) for p in params]
    plan = GradientTensors(grads, params=params, accums=accums)

    def double_step():
        leaves = [p.double().requires_grad_() for p in params]
        g1, b1, w, g2, b2, vv = leaves

        def norm(t, g, b):
            mu = t.mean(1, keepdim=True)
            return (t - mu) * ((t - mu).square().mean(1, keepdim=True) + 1e-3).rsqrt() * g + b
        s = norm(torch.tanh(norm(x.double(), g1, b1) @ w), g2, b2) @ vv
        logp = torch.log_softmax(s.view(B, L), 1)
        d = torch.autograd.grad(-(clicks.double() * logp).sum(), leaves)
        return ref_update([t for t in d], params, accums, 1.0 / B, 0.0, clip, lr, True)

    for _ in range(4):
        norm, ref = double_step()
        h0, s0 = layer_norm(x, params[0], params[1])
        a = torch.tanh(h0 @ params[2])
        h1, s1 = layer_norm(a, params[3], params[4])
        scores = (h1 @ params[5]).view(B, L)
        d_s = (torch.softmax(scores, 1) * clicks.sum(1, keepdim=True) - clicks).view(-1, 1)
        torch.mm(h1.t(), d_s, out=grads[5])
        d_a, _, _ = layer_norm_backward(d_s @ params[5].t(), a, s1, params[3], d_gamma=grads[3], d_beta=grads[4])
        d_z = d_a * (1 - a * a)
        torch.mm(h0.t(), d_z, out=grads[2])
        layer_norm_backward(d_z @ params[2].t(), x, s0, params[0], d_gamma=grads[0], d_beta=grads[1], need=(False, True, True))
        got = plan.clip_adagrad(clip, lr, scale=1.0 / B)
        # fp32 sums over 640 rows and 136 columns: 1e-4 of the largest step a parameter takes (lr / sqrt(0.1) * |e|) covers them
        assert abs(float(got) - norm) <= 1e-5 * norm
        for p, (rp, _, _, _) in zip(params, ref):
            assert (p.double() - rp).abs().max() <= 1e-5 * lr / 0.1 ** 0.5 + 2 * U


def test_lists_larger_than_the_last_level_cache():
    """Beyond 64 M elements the passes send data past the caches: same results."""
    from ultra_amd.learning_algorithm import GradientTensors
    sizes = [70000003, 5, 4097, 0, 8195]
    grads, params = tensors(sizes, (BF16, F32), 1, aligned=False), tensors(sizes, (F32,), 2, aligned=False)
    accums = [t.abs().add_(0.1) for t in tensors(sizes, (F32,), 3)]
    copies = tensors(sizes, (F16, BF16), 4, aligned=False)
    norm, ref = ref_update(grads, params, accums, 0.5, 0.01, 3.0, 0.05, True)
    plan = GradientTensors(grads, out=[torch.empty_like(g) for g in grads], params=params, accums=accums, copies=copies)
    out, plain = plan.clip(3.0, scale=0.5)
    want = 0.5 * ref_norm(grads)
    assert abs(float(plain) - want) <= 4 * U * want
    for o, g in zip(out, grads):
        w = g.double() * 0.5 * (3.0 / want)
        within(o, w, 5 * U * w.abs() + half_step(g.dtype, w), 'out')
    got = plan.clip_adagrad(3.0, 0.05, scale=0.5, l2=0.01)
    assert abs(float(got) - norm) <= 8 * U * norm
    for p, a, c, (rp, tp, ra, ta) in zip(params, accums, copies, ref):
        within(p, rp, tp, 'param')
        within(a, ra, ta, 'accum')
        assert torch.equal(c, p.to(c.dtype))
