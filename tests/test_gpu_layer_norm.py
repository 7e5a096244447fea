"""GPU tests (-m gpu) of the stand-alone layer norm, forward and backward, against its formulas in 64 bits.

Tolerances, per element.  u = 2^-24 is half a step of fp32, h(t) = finfo(t).eps / 2 half a step of the stored type.  A sum over
N entries runs through at most N / 64 + 32 additions in a row (64 lanes or more share a row), so its error is at most
(N / 64 + 32) u sum|.|; the elementwise arithmetic adds a few u.  A sum over M rows: at most M / 8 + 160 in a row."""
import itertools

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float32), (torch.float16, torch.float16)]
EPS = 1e-3


def half_step(t, v):
    f = torch.finfo(t)
    return f.eps / 2 * v.abs() + f.smallest_normal * f.eps / 2


def rows(m, n, dtype, seed, gap=0, shift=0, scale=1.0, offset=0.0):
    """[m, n] inside a buffer of its own: rows gap elements further apart, the first one shift elements in."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    buf = torch.full((m * (n + gap) + shift,), 7.0, dtype=dtype, device='cuda')
    t = buf[shift:].view(m, n + gap)[:, :n]
    t.copy_(torch.randn((m, n), generator=g, device='cuda') * scale + offset)
    return t, buf


def weights(n, dtype, seed, which=3):
    g = torch.Generator(device='cuda').manual_seed(seed)
    gamma = (1 + 0.3 * torch.randn(n, generator=g, device='cuda')).to(dtype)
    beta = torch.randn(n, generator=g, device='cuda').to(dtype)
    return gamma if which & 1 else None, beta if which & 2 else None


def ref_forward(x, gamma, beta, eps=EPS):
    """y, stats, and the tolerance of each."""
    xd = x.double()
    n = x.shape[-1]
    g = torch.ones(n, dtype=torch.float64, device='cuda') if gamma is None else gamma.double()
    b = torch.zeros(n, dtype=torch.float64, device='cuda') if beta is None else beta.double()
    mean = xd.mean(-1, keepdim=True)
    var = (xd - mean).square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    xh = (xd - mean) * rstd
    y = xh * g + b
    d = n / 64 + 32
    dmean = (d + 1) * U * xd.abs().mean(-1, keepdim=True)
    # the variance: d + 4 roundings of positive terms, and the mean's error enters squared and through the terms' rounding
    rel = ((d + 6) * U * var + dmean ** 2 + 4 * U * dmean * var.sqrt()) / (var + eps) / 2 + 4 * U
    tol_y = half_step(x.dtype, y) + g.abs() * rstd * dmean + (xh * g).abs() * (rel + 4 * U) + U * (y.abs() + (xh * g).abs())
    tol_s = torch.cat([dmean + U * mean.abs(), rstd * rel], -1)
    return y, torch.cat([mean, rstd], -1), tol_y, tol_s


def ref_backward(dy, x, stats, gamma):
    n, m = x.shape[-1], x.numel() // x.shape[-1]
    g = torch.ones(n, dtype=torch.float64, device='cuda') if gamma is None else gamma.double()
    dyd, mean, rstd = dy.double(), stats[..., :1].double(), stats[..., 1:].double()
    xh = (x.double() - mean) * rstd
    gr = dyd * g
    a, b = gr.mean(-1, keepdim=True), (gr * xh).mean(-1, keepdim=True)
    dx = rstd * (gr - a - xh * b)
    d = n / 64 + 32
    tol = half_step(x.dtype, dx) + rstd * U * (8 * gr.abs() + (d + 8) * gr.abs().mean(-1, keepdim=True) +
                                               (d + 16) * xh.abs() * (gr * xh).abs().mean(-1, keepdim=True))
    dims = tuple(range(x.dim() - 1))
    r = m / 8 + 160
    dg, db = (dyd * xh).sum(dims), dyd.sum(dims)
    tol_g, tol_b = (r + 4) * U * (dyd * xh).abs().sum(dims), r * U * dyd.abs().sum(dims)
    return dx, dg, db, tol, tol_g, tol_b


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    if bad.any():
        k = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError('%s: %d of %d off, first at %d: got %r want %r tol %r' % (
            what, int(bad.sum()), bad.numel(), k, got.reshape(-1)[k].item(), want.reshape(-1)[k].item(), tol.reshape(-1)[k].item()))


SIZES = [(1, 1), (3, 1), (1, 2), (2, 3), (2, 7), (5, 8), (9, 15), (7, 33), (64, 63), (4, 64), (33, 65), (10, 136), (17, 255), (6, 256),
         (9, 700), (3, 1023), (2, 1024), (5, 1025), (3, 2047), (3, 2048), (3, 2049), (2, 4096), (2, 4099), (2, 5003), (2, 8192),
         (1, 8193), (2, 12345), (2, 16384), (2, 16385), (1, 32768), (1, 32769), (2, 65535), (1, 65536),
         (5, 40), (5, 57), (5, 100), (5, 200), (5, 400), (3, 900), (3, 1592), (3, 3300), (3, 3585)]


@pytest.mark.parametrize('m,n', SIZES)
def test_forward_widths(m, n):
    from ultra_amd.ranking_model import layer_norm
    for k, (t, w) in enumerate(TYPES):
        x, _ = rows(m, n, t, k, scale=1.5, offset=0.7)
        gamma, beta = weights(n, w, k + 10, which=(3, 1, 2, 0, 3)[k] if n % 2 else 3)
        y, stats = layer_norm(x, gamma, beta)
        ry, rs, ty, ts = ref_forward(x, gamma, beta)
        within(stats, rs, ts, 'stats %s' % t)
        within(y, ry, ty, 'y %s %s' % (t, w))


@pytest.mark.parametrize('m', [1, 2, 3, 4, 5, 31, 255, 256, 257, 4097, 70001])
@pytest.mark.parametrize('n', [1, 10, 136])
def test_forward_many_rows(m, n):
    from ultra_amd.ranking_model import layer_norm
    for k, (t, w) in enumerate(TYPES[::2]):
        x, _ = rows(m, n, t, k)
        gamma, beta = weights(n, w, k)
        y, stats = layer_norm(x, gamma, beta)
        ry, rs, ty, ts = ref_forward(x, gamma, beta)
        within(stats, rs, ts, 'stats')
        within(y, ry, ty, 'y')


LAYOUTS = [(0, 1), (1, 0), (3, 1), (5, 3), (8, 2), (64, 0)]  # (elements between rows, elements before the first)


@pytest.mark.parametrize('gap,shift', LAYOUTS)
@pytest.mark.parametrize('n', [1, 6, 136, 700, 1025, 5003])
def test_forward_layouts_leave_the_rest_alone(gap, shift, n):
    from ultra_amd.ranking_model import layer_norm
    for k, (t, w) in enumerate(TYPES):
        x, _ = rows(11, n, t, k, gap, shift)
        gw, bw = rows(1, n, w, 5, 0, shift)[0][0], rows(1, n, w, 6, 0, (shift * 3) % 4)[0][0]
        y, buf = rows(11, n, t, 99, gap, shift)
        before = buf.clone()
        layer_norm(x, gw, bw, out=y)
        ry, _, ty, _ = ref_forward(x, gw, bw)
        within(y, ry, ty, 'y')
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[shift:].view(11, n + gap)[:, :n] = False
        assert torch.equal(buf[keep], before[keep])


def test_forward_in_place_and_batched_shapes():
    from ultra_amd.ranking_model import layer_norm
    for n, (t, w) in itertools.product((7, 136, 4096, 5003), TYPES):
        x, _ = rows(12, n, t, 3)
        gamma, beta = weights(n, w, 4)
        ry, _, ty, _ = ref_forward(x, gamma, beta)
        z = x.clone().view(3, 4, n)
        y, stats = layer_norm(z, gamma, beta, out=z)
        assert y is z and stats.shape == (3, 4, 2)
        within(y.view(12, n), ry, ty, 'in place')
    table, _ = rows(12, 40, torch.float32, 1)
    view = table.view(3, 4, 40)[:, :, 5:30]  # a slice of a table: one stride for all rows
    y, _ = layer_norm(view)
    ry, _, ty, _ = ref_forward(view, None, None)
    within(y, ry, ty, 'slice')
    one = torch.randn(9, device='cuda')
    y, stats = layer_norm(one)
    assert y.shape == (9,) and stats.shape == (2,)
    within(y, ref_forward(one, None, None)[0], ref_forward(one, None, None)[2], 'a vector')


@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16, torch.float16])
def test_rows_without_variance_and_far_from_zero(t):
    from ultra_amd.ranking_model import layer_norm
    for n in (1, 5, 136, 1024, 5003):
        x = torch.full((3, n), 2.5, dtype=t, device='cuda')
        x[1] = 0
        x[2] = -1000.0
        gamma, beta = weights(n, torch.float32, 1)
        y, stats = layer_norm(x, gamma, beta)
        ry, rs, ty, ts = ref_forward(x, gamma, beta)
        within(y, ry, ty, 'constant')
        within(stats, rs, ts, 'constant stats')
        x, _ = rows(3, n, t, 2, scale=0.5, offset=300.0)
        y, stats = layer_norm(x, gamma, beta)
        ry, rs, ty, ts = ref_forward(x, gamma, beta)
        within(y, ry, ty, 'offset')
        within(stats, rs, ts, 'offset stats')


@pytest.mark.parametrize('n', [8, 136, 2049, 5003, 40000])
def test_a_bad_row_stays_alone(n):
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    for t in (torch.float32, torch.bfloat16, torch.float16):
        x, _ = rows(9, n, t, 3)
        clean, cs = layer_norm(x)
        for k, bad in enumerate((float('nan'), float('inf'), float('-inf'))):
            z = x.clone()
            z[4, (k * 7919) % n] = bad
            y, stats = layer_norm(z)
            assert torch.isnan(y[4]).all() and torch.isnan(stats[4, 1])
            others = [r for r in range(9) if r != 4]
            assert torch.equal(y[others], clean[others]) and torch.equal(stats[others], cs[others])
            dx, _, _ = layer_norm_backward(x, z, stats, need=(True, False, False))
            assert torch.isnan(dx[4]).all() and torch.isfinite(dx[others]).all()


def test_no_rows():
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    x = torch.empty((0, 136), device='cuda')
    y, stats = layer_norm(x)
    assert y.shape == (0, 136) and stats.shape == (0, 2)
    dg, db = torch.full((136,), 5.0, device='cuda'), torch.full((136,), 5.0, device='cuda')
    layer_norm_backward(x, x.clone(), stats, d_gamma=dg, d_beta=db)
    assert not dg.any() and not db.any()


@pytest.mark.parametrize('m,n', SIZES + [(257, 1), (300, 17), (70, 136), (4097, 10), (1000, 512), (70001, 3), (2050, 136), (513, 1500),
                                         (130, 4096), (600, 5003),
                                         # on both sides of where the pass changes: 512 and 1024 rows, 8192 and 32768 entries
                                         (512, 1100), (513, 1100), (512, 8192), (513, 8192), (700, 8193), (1024, 8200), (1025, 8200),
                                         (1030, 9001), (2100, 9000), (40, 32768), (40, 33001), (600, 33001)])
def test_backward(m, n):
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    for k, (t, w) in enumerate(TYPES):
        x, _ = rows(m, n, t, k, scale=1.5, offset=0.4)
        dy, _ = rows(m, n, t, k + 50)
        gamma, _ = weights(n, w, k)
        if n % 5 == 0 and k < 2:
            gamma = None
        _, stats = layer_norm(x, gamma)
        dx, dg, db = layer_norm_backward(dy, x, stats, gamma)
        rx, rg, rb, tx, tg, tb = ref_backward(dy, x, stats, gamma)
        within(dx, rx, tx, 'dx %s' % t)
        within(dg, rg, tg + half_step(dg.dtype, rg), 'd_gamma %s' % w)
        within(db, rb, tb + half_step(db.dtype, rb), 'd_beta %s' % w)
        # the same call gives the same bits, and each part alone what all give together
        again = layer_norm_backward(dy, x, stats, gamma)
        assert all(torch.equal(p, q) for p, q in zip((dx, dg, db), again))
        ex = layer_norm_backward(dy, x, stats, gamma, need=(True, False, False))
        assert ex[1] is None and ex[2] is None
        within(ex[0], rx, tx, 'dx alone')
        eg = layer_norm_backward(dy, x, stats, gamma, need=(False, True, False))
        assert eg[0] is None and eg[2] is None
        within(eg[1], rg, tg + half_step(dg.dtype, rg), 'd_gamma alone')
        eb = layer_norm_backward(dy, x, stats, gamma, need=(False, False, True))
        within(eb[2], rb, tb + half_step(eb[2].dtype, rb), 'd_beta alone')


@pytest.mark.parametrize('gap,shift', LAYOUTS)
@pytest.mark.parametrize('m,n', [(11, 1), (11, 6), (300, 136), (37, 700), (11, 1025), (700, 1025), (11, 5003)])
def test_backward_layouts_leave_the_rest_alone(gap, shift, m, n):
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    for k, (t, w) in enumerate(TYPES):
        x, _ = rows(m, n, t, k, gap, shift)
        dy, _ = rows(m, n, t, k + 9, (gap * 3) % 7, (shift + 1) % 3)
        gamma = rows(1, n, w, 5, 0, shift)[0][0]
        dx, buf = rows(m, n, t, 99, gap, shift)
        dgb, dbb = (torch.full((n + 8,), 3.0, dtype=w, device='cuda') for _ in range(2))
        dg, db = dgb[shift:shift + n], dbb[3:3 + n]
        before = buf.clone()
        _, stats = layer_norm(x)
        layer_norm_backward(dy, x, stats, gamma, d_x=dx, d_gamma=dg, d_beta=db)
        rx, rg, rb, tx, tg, tb = ref_backward(dy, x, stats, gamma)
        within(dx, rx, tx, 'dx')
        within(dg, rg, tg + half_step(w, rg), 'd_gamma')
        within(db, rb, tb + half_step(w, rb), 'd_beta')
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[shift:].view(m, n + gap)[:, :n] = False
        assert torch.equal(buf[keep], before[keep])
        assert (dgb[:shift] == 3).all() and (dgb[shift + n:] == 3).all() and (dbb[:3] == 3).all() and (dbb[3 + n:] == 3).all()


def test_backward_is_the_forward_passes_difference():
    """Central differences of the formula in 64 bits: truncation error O(step^2) with third derivatives of order one."""
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    m, n, step = 3, 9, 1e-5
    x, _ = rows(m, n, torch.float32, 1)
    c, _ = rows(m, n, torch.float32, 2)
    gamma, beta = weights(n, torch.float32, 3)
    _, stats = layer_norm(x, gamma, beta)
    dx, dg, db = layer_norm_backward(c, x, stats, gamma)

    def loss(xv, gv, bv):
        mu = xv.mean(1, keepdims=True)
        return float((((xv - mu) / np.sqrt(((xv - mu) ** 2).mean(1, keepdims=True) + EPS) * gv + bv) * c.double().cpu().numpy()).sum())
    args = [v.double().cpu().numpy() for v in (x, gamma, beta)]
    for which, got in enumerate((dx, dg, db)):
        want = np.zeros(args[which].shape)
        for idx in np.ndindex(want.shape):
            lo, hi = [a.copy() for a in args], [a.copy() for a in args]
            lo[which][idx] -= step
            hi[which][idx] += step
            want[idx] = (loss(*hi) - loss(*lo)) / (2 * step)
        assert np.abs(got.double().cpu().numpy() - want).max() < 2e-5


def test_rows_beyond_32_bit_offsets():
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    n, ld = 1000, (1 << 30) + 77
    buf = torch.zeros(2 * ld + n, dtype=torch.bfloat16, device='cuda')  # 4.3 GB: the last row starts beyond 2^31 elements
    x = buf.as_strided((3, n), (ld, 1))
    x.copy_(rows(3, n, torch.bfloat16, 1)[0])
    y, stats = layer_norm(x, out=None)
    ry, rs, ty, ts = ref_forward(x, None, None)
    within(y, ry, ty, 'y')
    dx, dg, db = layer_norm_backward(x, x, stats)
    rx, rg, rb, tx, tg, tb = ref_backward(x, x, stats, None)
    within(dx, rx, tx, 'dx')
    within(dg, rg, tg, 'd_gamma')
    out = torch.zeros_like(buf).as_strided((3, n), (ld, 1))
    layer_norm(x, out=out)
    assert torch.equal(out, y)


def test_more_rows_than_one_grid_takes():
    from ultra_amd.ranking_model import layer_norm
    m = (1 << 27) + (1 << 20) + 5
    x = torch.randn((m, 2), device='cuda', dtype=torch.float16)
    y, stats = layer_norm(x)
    for at in (0, (1 << 27) - 300, m - 300):
        part = slice(at, min(m, at + 700))
        ry, rs, ty, ts = ref_forward(x[part], None, None)
        within(y[part], ry, ty, 'y')
        within(stats[part], rs, ts, 'stats')
    assert torch.isfinite(stats).all()


def test_streams_and_workspaces():
    """Two backward passes in flight, each with its own workspace, on streams of their own."""
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward, layer_norm_workspace
    m, n = 3000, 1030
    jobs = []
    for k in range(2):
        x, dy = rows(m, n, torch.bfloat16, k)[0], rows(m, n, torch.bfloat16, k + 7)[0]
        gamma, _ = weights(n, torch.float32, k)
        _, stats = layer_norm(x)
        jobs.append((dy, x, stats, gamma, layer_norm_workspace(m, n, 'cuda'), layer_norm_backward(dy, x, stats, gamma)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(3):
        for s, (dy, x, stats, gamma, ws, _) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(layer_norm_backward(dy, x, stats, gamma, workspace=ws))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, jobs[k % 2][5]))


@pytest.mark.parametrize('m,n', [(5, 136), (3000, 700), (64, 5003), (1100, 8200)])
def test_captured_and_replayed(m, n):
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward, layer_norm_workspace
    x, dy = rows(m, n, torch.float32, 1)[0], rows(m, n, torch.float32, 2)[0]
    gamma, beta = weights(n, torch.float32, 3)
    y, stats, dx = torch.empty_like(x), torch.empty((m, 2), device='cuda'), torch.empty_like(x)
    dg, db, ws = torch.empty_like(gamma), torch.empty_like(gamma), layer_norm_workspace(m, n, 'cuda')

    def step():
        layer_norm(x, gamma, beta, out=y, stats=stats)
        layer_norm_backward(dy, x, stats, gamma, d_x=dx, d_gamma=dg, d_beta=db, workspace=ws)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        x.copy_(rows(m, n, torch.float32, 20 + k)[0])
        dy.copy_(rows(m, n, torch.float32, 30 + k)[0])
        ws.fill_(255)  # NaN: nothing of the workspace is read before it is written
        graph.replay()
        got = [t.clone() for t in (y, stats, dx, dg, db)]
        torch.cuda.synchronize()
        step()
        assert all(torch.equal(p, q) for p, q in zip(got, (y, stats, dx, dg, db)))
        torch.cuda.synchronize()


def test_what_the_c_call_leaves_out():
    """No statistics, no weights, one row whose stride is nonsense, no workspace where none is needed."""
    from ultra_amd import _lib
    lib, st = _lib.lib(), _lib.current_stream()
    x, _ = rows(1, 700, torch.float16, 1)
    gamma, _ = weights(700, torch.float16, 2)
    y = torch.empty_like(x)
    for ld in (0, -5, 3, 1 << 39):
        y.fill_(0)
        assert lib.ultr_layer_norm_forward(x.data_ptr(), ld, gamma.data_ptr(), None, 1, 700, EPS, _lib.DTYPE_F16, _lib.DTYPE_F16,
                                           y.data_ptr(), ld, None, st) == 0
        ry, rs, ty, _ = ref_forward(x, gamma, None)
        within(y, ry, ty, 'y')
    stats = rs.float()
    dx, db = torch.empty_like(x), torch.empty(700, dtype=torch.float16, device='cuda')
    assert lib.ultr_layer_norm_workspace_bytes(1, 700) == 0
    assert lib.ultr_layer_norm_backward(y.data_ptr(), 0, x.data_ptr(), -1, stats.data_ptr(), None, 1, 700, _lib.DTYPE_F16, _lib.DTYPE_F16,
                                        dx.data_ptr(), 0, None, db.data_ptr(), None, st) == 0
    rx, _, rb, tx, _, tb = ref_backward(y, x, stats, None)
    within(dx, rx, tx, 'dx')
    within(db, rb, tb + half_step(torch.float16, rb), 'd_beta')
    # no rows: weight gradients are zero, nothing else is touched
    db.fill_(3)
    assert lib.ultr_layer_norm_backward(None, 0, None, 0, None, None, 0, 700, _lib.DTYPE_F16, _lib.DTYPE_F16, None, 0, None, db.data_ptr(),
                                        None, st) == 0
    assert not db.any()


def test_python_refusals():
    from ultra_amd import _lib
    from ultra_amd.ranking_model import layer_norm, layer_norm_backward
    x = torch.randn((4, 6, 8), device='cuda')
    for bad in (torch.randn(4, 8), x.double(), x.transpose(1, 2), x.transpose(0, 1), torch.empty((4, 0), device='cuda'),
                torch.tensor(1.0, device='cuda')):
        with pytest.raises(ValueError):
            layer_norm(bad)
    with pytest.raises(_lib.UltrError):
        layer_norm(torch.randn(8, device='cuda').expand(4, 8), out=torch.empty((4, 8), device='cuda'))  # rows on one another
    g = torch.ones(8, device='cuda')
    for kw in (dict(gamma=g[:7]), dict(gamma=g.half()), dict(gamma=g.cpu()), dict(beta=torch.ones(16, device='cuda')[::2]),
               dict(out=x[:2]), dict(out=x.half()), dict(stats=torch.empty((4, 6), device='cuda'))):
        with pytest.raises(ValueError):
            layer_norm(x, **kw)
    h = x.half()
    with pytest.raises(ValueError):
        layer_norm(h, gamma=g, beta=g.half())
    _, stats = layer_norm(x)
    with pytest.raises(ValueError):
        layer_norm_backward(x[:2], x, stats)
    with pytest.raises(ValueError):
        layer_norm_backward(x, x, stats[:2])
    with pytest.raises(_lib.UltrError):
        layer_norm_backward(x, x, stats, d_x=x)
    with pytest.raises(_lib.UltrError):
        layer_norm_backward(x, x, stats, need=(False, False, False))
    wide = torch.randn((900, 4096), device='cuda')
    _, ws_stats = layer_norm(wide)
    with pytest.raises(ValueError):
        layer_norm_backward(wide, wide, ws_stats, workspace=torch.empty(16, dtype=torch.uint8, device='cuda'))
