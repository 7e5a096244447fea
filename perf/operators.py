"""Workloads for the stand-alone operators: layer norm (forward, backward), the global gradient norm with clipping over
many tensors, and the clipped optimiser update over many tensors.

``own`` False: every operator in its plain form, elementary torch operations in 32 bits, rounded once at the end.
``own`` True: the calls a user makes of ``ultra_amd``.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math
import zlib

import torch

own = False

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2, 'none': 0}
EPS = 1e-3           # the framework's layer normalisation epsilon
MOST_NORM = 16384 * 4096
MOST_CLIP = 600 * 10**6
MOST_UPDATE = 200 * 10**6


def listed():
    return [
        # one row through a 512-wide layer, as when a single document is scored: nothing but latency
        {'name': 'norm, one row', 'op': 'norm', 'rows': 1, 'cols': 512, 'gap': 0, 'dtype': 'f32', 'wdtype': 'f32'},
        # a wide odd row out of a wider table (row stride beyond the width), half precision
        {'name': 'norm, odd rows in a table', 'op': 'norm', 'rows': 3001, 'cols': 5003, 'gap': 13, 'dtype': 'f16', 'wdtype': 'f32'},
        # a training batch of a large model, everything in bfloat16
        {'name': 'norm, large batch', 'op': 'norm', 'rows': 16384, 'cols': 4096, 'gap': 0, 'dtype': 'bf16', 'wdtype': 'bf16'},
        # the gradient of one list of 10 documents with 136 features
        {'name': 'norm gradient, one list', 'op': 'norm_grad', 'rows': 10, 'cols': 136, 'gap': 0, 'dtype': 'f32', 'wdtype': 'f32'},
        # 4096 lists of 10 documents at the first hidden layer: many rows, narrow, the weight gradient sums 40960 of them
        {'name': 'norm gradient, 4096 lists', 'op': 'norm_grad', 'rows': 40960, 'cols': 512, 'gap': 0, 'dtype': 'f32', 'wdtype': 'f32'},
        # few very wide odd rows
        {'name': 'norm gradient, odd wide rows', 'op': 'norm_grad', 'rows': 777, 'cols': 12345, 'gap': 0, 'dtype': 'bf16', 'wdtype': 'f32'},
        # the large batch's backward pass
        {'name': 'norm gradient, large batch', 'op': 'norm_grad', 'rows': 16384, 'cols': 4096, 'gap': 0, 'dtype': 'bf16', 'wdtype': 'f32'},
        # the default scorer's 16 variables at 136 features
        {'name': 'clip, default scorer', 'op': 'clip', 'sizes': 'mlp', 'count': 136, 'width': 512, 'dtype': 'f32', 'clip': 5.0},
        # a thousand ragged tensors of all sizes (tables, biases, scalars): none aligned with the next
        {'name': 'clip, ragged tensors', 'op': 'clip', 'sizes': 'ragged', 'count': 1000, 'width': 60000, 'dtype': 'f32', 'clip': 1.0},
        # a large model's gradients in bfloat16
        {'name': 'clip, large model', 'op': 'clip', 'sizes': 'blocks', 'count': 11, 'width': 2048, 'dtype': 'bf16', 'clip': 1.0},
        # the default scorer's update at 700 features
        {'name': 'update, default scorer', 'op': 'update', 'sizes': 'mlp', 'count': 700, 'width': 512, 'dtype': 'f32', 'copy': 'none', 'clip': 5.0},
        # a large model's update: bfloat16 gradients, 32-bit masters and accumulators, bfloat16 copies written on the way
        {'name': 'update, large model', 'op': 'update', 'sizes': 'blocks', 'count': 3, 'width': 2048, 'dtype': 'bf16', 'copy': 'bf16', 'clip': 1.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(('norm', 'norm_grad', 'clip', 'update'))
    dtype = rng.choice(('f32', 'bf16', 'f16'))
    if op in ('norm', 'norm_grad'):
        cols = _spread(rng, 8, 65536)
        # 32-bit types move twice the bytes of the largest listed case per element
        rows = _spread(rng, 1, max(2, min(131072, MOST_NORM // (2 * cols))))
        return {'op': op, 'rows': rows, 'cols': cols, 'gap': rng.choice((0, 0, rng.randint(1, 64))), 'dtype': dtype,
                'wdtype': rng.choice(('f32', dtype))}
    most = (MOST_CLIP if op == 'clip' else MOST_UPDATE) // 2
    kind = rng.choice(('mlp', 'ragged', 'blocks'))
    if kind == 'mlp':
        count, width = _spread(rng, 16, 4096), _spread(rng, 8, 4096)
    elif kind == 'ragged':
        count = _spread(rng, 1, 3000)
        width = _spread(rng, 16, min(4 * 10**6, 8 * most // count))
    else:
        width = _spread(rng, 32, 2048)
        count = rng.randint(1, max(1, min(24, most // (12 * width * width + 7 * width))))
    case = {'op': op, 'sizes': kind, 'count': count, 'width': width, 'dtype': dtype, 'clip': rng.choice((0.5, 1.0, 5.0))}
    if dtype == 'f16':  # gradients scaled for a type of little range, and a bound to match: clipped ones keep their bits
        case['clip'] = round(rng.uniform(0.1, 1.0) * math.sqrt(sum(_shapes(case))), 3)
    if op == 'update':
        case['copy'] = rng.choice(('none', 'bf16', 'f16'))
    return case


def _shapes(case):
    """Elements of each tensor: from the case alone."""
    n, w = case['count'], case['width']
    if case['sizes'] == 'mlp':  # n features into layers of w, w / 2, w / 4 and one score: W, b, gamma, beta of each
        widths = [n, w, max(1, w // 2), max(1, w // 4), 1]
        return [s for k, m in zip(widths, widths[1:]) for s in (k * m, m, k, k)]
    if case['sizes'] == 'blocks':  # n blocks: four square matrices, two of four times the width, and their vectors
        return [w * w, w] * (4 * n) + [4 * w * w, w] * n + [4 * w * w, 2 * w] * n
    return [1 + int(w ** ((zlib.crc32(b'%d' % i) % 10007) / 10007.0)) for i in range(n)]  # 'ragged': 2 to w + 1, over the logarithm


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _rows(g, case, scale, shift):
    """[rows, cols] inside a table whose rows are ``gap`` elements further apart."""
    m, n = case['rows'], case['cols']
    t = torch.randn((m, n + case['gap']), generator=g, device='cuda')
    if scale is not None:
        t = t * scale + shift
    return t.to(DTYPES[case['dtype']])[:, :n]


def _weights(g, case):
    n, w = case['cols'], DTYPES[case['wdtype']]
    gamma = (1 + 0.2 * torch.randn(n, generator=g, device='cuda')).to(w)
    beta = (0.2 * torch.randn(n, generator=g, device='cuda')).to(w)
    return gamma, beta


def prepare(case, seed):
    g = _generator(seed)
    if case['op'] in ('norm', 'norm_grad'):
        m, n = case['rows'], case['cols']
        # rows of different scale and offset, as activations have
        scale = 0.5 + 2 * torch.rand((m, 1), generator=g, device='cuda')
        s = {'case': case, 'x': _rows(g, case, scale, 2 * torch.randn((m, 1), generator=g, device='cuda'))}
        s['gamma'], s['beta'] = _weights(g, case)
        if case['op'] == 'norm':
            s['y'] = torch.empty((m, n), dtype=s['x'].dtype, device='cuda')
            s['stats'] = torch.empty((m, 2), device='cuda')
            return s
        s['dy'] = _rows(g, case, None, None)
        s['stats'] = _statistics(s['x'].float())
        s['dx'] = torch.empty((m, n), dtype=s['x'].dtype, device='cuda')
        s['dgamma'], s['dbeta'] = torch.empty_like(s['gamma']), torch.empty_like(s['beta'])
        if own:
            from ultra_amd.ranking_model import layer_norm_workspace
            s['ws'] = layer_norm_workspace(m, n, s['x'].device)
        return s
    shapes = _shapes(case)
    total = sum(shapes)
    # gradients of very different size per tensor; each tensor has its own storage
    grads = [t.clone() for t in torch.randn(total, generator=g, device='cuda').to(DTYPES[case['dtype']]).split(shapes)]
    for k, t in enumerate(grads):
        t.mul_(10.0 ** -(k % 4))
    s = {'case': case, 'grads': grads}
    if case['op'] == 'clip':
        s['out'] = torch.empty(total, dtype=grads[0].dtype, device='cuda')
        if own:
            from ultra_amd.learning_algorithm import GradientTensors
            s['plan'] = GradientTensors(grads, out=list(s['out'].split(shapes)))
        return s
    s['denom'] = torch.full((1,), 64.0, device='cuda')  # the batch's normaliser, known on the device only
    s['params'] = 0.05 * torch.randn(total, generator=g, device='cuda')
    s['accums'] = torch.full((total,), 0.1, device='cuda')
    s['copy'] = torch.empty(total, dtype=DTYPES[case['copy']], device='cuda') if case['copy'] != 'none' else None
    if own:
        from ultra_amd.learning_algorithm import GradientTensors
        s['plan'] = GradientTensors(grads, params=list(s['params'].split(shapes)), accums=list(s['accums'].split(shapes)),
                                    copies=None if s['copy'] is None else list(s['copy'].split(shapes)))
    return s


def _statistics(x):
    mean = x.mean(dim=1, keepdim=True)
    var = (x - mean).square().mean(dim=1, keepdim=True)
    return torch.cat([mean, torch.rsqrt(var + EPS)], dim=1)


LR = 0.05


def run(s):
    case = s['case']
    if own:
        return _run_own(s, case['op'])
    if case['op'] == 'norm':
        x = s['x'].float()
        stats = _statistics(x)
        y = (x - stats[:, :1]) * stats[:, 1:] * s['gamma'].float() + s['beta'].float()
        return {'y': y.to(s['x'].dtype), 'stats': stats}
    if case['op'] == 'norm_grad':
        dy, rstd = s['dy'].float(), s['stats'][:, 1:]
        xhat = (s['x'].float() - s['stats'][:, :1]) * rstd
        gr = dy * s['gamma'].float()
        dx = rstd * (gr - gr.mean(dim=1, keepdim=True) - xhat * (gr * xhat).mean(dim=1, keepdim=True))
        return {'dx': dx.to(s['x'].dtype), 'dgamma': (dy * xhat).sum(dim=0).to(s['gamma'].dtype),
                'dbeta': dy.sum(dim=0).to(s['beta'].dtype)}
    flat = torch.cat(s['grads']).float()
    if case['op'] == 'clip':
        norm = flat.square().sum().sqrt().view(1)
        return {'out': (flat * (case['clip'] / norm.clamp_min(case['clip']))).to(s['out'].dtype), 'norm': norm}
    flat = flat / s['denom']
    norm = flat.square().sum().sqrt().view(1)
    flat = flat * (case['clip'] / norm.clamp_min(case['clip']))
    s['accums'].add_(flat.square())
    s['params'].sub_(LR * flat / s['accums'].sqrt())
    out = {'params': s['params'], 'accums': s['accums'], 'norm': norm}
    if s['copy'] is not None:
        s['copy'].copy_(s['params'])
        out['copy'] = s['copy']
    return out


def _run_own(s, op):
    case = s['case']
    if op == 'norm':
        from ultra_amd.ranking_model import layer_norm
        y, stats = layer_norm(s['x'], s['gamma'], s['beta'], eps=EPS, out=s['y'], stats=s['stats'])
        return {'y': y, 'stats': stats}
    if op == 'norm_grad':
        from ultra_amd.ranking_model import layer_norm_backward
        dx, dgamma, dbeta = layer_norm_backward(s['dy'], s['x'], s['stats'], s['gamma'], d_x=s['dx'], d_gamma=s['dgamma'],
                                                d_beta=s['dbeta'], workspace=s['ws'])
        return {'dx': dx, 'dgamma': dgamma, 'dbeta': dbeta}
    if op == 'clip':
        _, norm = s['plan'].clip(case['clip'])
        return {'out': s['out'], 'norm': norm}
    norm = s['plan'].clip_adagrad(case['clip'], LR, denom=s['denom'])
    out = {'params': s['params'], 'accums': s['accums'], 'norm': norm}
    if s['copy'] is not None:
        out['copy'] = s['copy']
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'norm':
        x = s['x'].double()
        centred = x - x.mean(dim=1, keepdim=True)
        rstd = (centred.pow(2).mean(dim=1, keepdim=True) + EPS).pow(-0.5)
        return {'y': centred * rstd * s['gamma'].double() + s['beta'].double(),
                'stats': torch.cat([x.mean(dim=1, keepdim=True), rstd], dim=1)}
    if case['op'] == 'norm_grad':
        dy, mean, rstd = s['dy'].double(), s['stats'][:, 0].double(), s['stats'][:, 1].double()
        xhat = (s['x'].double() - mean[:, None]) * rstd[:, None]
        gr, n = dy * s['gamma'].double(), case['cols']
        dx = rstd[:, None] * (gr - (gr.sum(dim=1) / n)[:, None] - xhat * ((gr * xhat).sum(dim=1) / n)[:, None])
        return {'dx': dx, 'dgamma': (dy * xhat).sum(dim=0), 'dbeta': dy.sum(dim=0)}
    flat = torch.cat(s['grads']).double()
    if case['op'] == 'update':
        flat = flat / 64
    norm = flat.pow(2).sum().sqrt()
    flat = flat * min(1.0, case['clip'] / float(norm))
    if case['op'] == 'clip':
        return {'out': flat, 'norm': norm.view(1)}
    accums = s['accums'].double() + flat.pow(2)
    params = s['params'].double() - LR * flat / accums.sqrt()
    out = {'params': params, 'accums': accums, 'norm': norm.view(1)}
    if case['copy'] != 'none':
        out['copy'] = params
    return out


def work(case):
    if case['op'] in ('norm', 'norm_grad'):
        m, n, e, w = case['rows'], case['cols'], BYTES[case['dtype']], BYTES[case['wdtype']]
        if case['op'] == 'norm':
            return {'bytes': 2 * m * n * e + 2 * n * w + 8 * m, 'flops': 8 * m * n}
        return {'bytes': 3 * m * n * e + 3 * n * w + 8 * m, 'flops': 16 * m * n}
    total, e = sum(_shapes(case)), BYTES[case['dtype']]
    if case['op'] == 'clip':
        return {'bytes': 2 * total * e + 4, 'flops': 3 * total}
    return {'bytes': total * (e + 16 + BYTES[case['copy']]) + 8, 'flops': 9 * total}
