"""Layer norm calls whose arguments share memory that one of them writes are refused on the host, before any launch.  No GPU
needed: the addresses are never touched.  (Calls that are accepted would launch: those are tested on the GPU.)"""
import random

import pytest

from tests.test_operator_refusals import F32, F16, P, backward, forward, last


@pytest.mark.parametrize('kw', [
    dict(gamma=2 * P), dict(beta=2 * P + 60), dict(gamma=2 * P - 28), dict(stats=P), dict(stats=P + 56), dict(stats=2 * P - 8),
    dict(gamma=3 * P, stats=3 * P + 8), dict(beta=3 * P, stats=3 * P - 8), dict(gamma=2 * P + 32, N=1), dict(y=P + 16, ldx=16, ldy=16),
    dict(y=P + 16 * 4 - 4, ldx=16, ldy=16), dict(y=P - 16, ldx=16, ldy=16), dict(ldx=1 << 39, y=P + (1 << 41), M=4, ldy=1 << 39),
    dict(x=P, ldx=20, y=P + 32, ldy=21),  # different strides: their ends are looked at, nothing else
])
def test_forward_refuses_shared_memory(kw):
    assert forward(**kw) == -1
    assert 'overlaps' in last()


@pytest.mark.parametrize('kw', [
    dict(dx=3 * P), dict(dx=3 * P - 60), dict(gamma=4 * P + 32), dict(dx=5 * P), dict(db=4 * P + 60), dict(dg=P + 60), dict(dg=2 * P - 28),
    dict(db=3 * P + 8), dict(dg=6 * P + 28), dict(dx=2 * P + 16, ldx=16, lddx=16), dict(dx=P - 32 + 64, lddy=16, lddx=16, xd=F32, dg=P),
    dict(M=3000, N=700, ldx=700, lddy=700, lddx=700, dy=P, x=100 * P, dx=200 * P, ws=200 * P + 64),
    dict(M=3000, N=700, ldx=700, lddy=700, lddx=700, dy=P, x=100 * P, dx=200 * P, ws=99 * P, xd=F16, wd=F16),
    dict(M=3000, N=700, ldx=700, lddy=700, lddx=700, dy=P, x=100 * P, dx=200 * P, dg=300 * P + 64, ws=300 * P, db=400 * P),
])
def test_backward_refuses_shared_memory(kw):
    assert backward(**kw) == -1
    assert 'overlaps' in last()


def rows_bytes(at, rows, ld, width):
    return {at + (r * ld + c) * 4 + b for r in range(rows) for c in range(width) for b in range(4)}


def test_every_shared_byte_is_found():
    """Random layouts against the sets of their bytes."""
    rng, met = random.Random(3), 0
    for _ in range(4000):
        m, n = rng.randint(1, 5), rng.randint(1, 6)
        ldx, ldy = n + rng.randint(0, 9), n + rng.randint(0, 9)
        if rng.random() < 0.6:
            ldy = ldx
        y = P + 4 * rng.randint(-60, 60)
        if y == P and (ldx == ldy or m == 1):  # in place
            continue
        stats = P + 8 * rng.randint(-40, 40)
        gamma = P + 4 * rng.randint(-60, 60)
        x_b, y_b = rows_bytes(P, m, ldx, n), rows_bytes(y, m, ldy, n)
        s_b, g_b = rows_bytes(stats, 1, 0, 2 * m), rows_bytes(gamma, 1, 0, n)
        kw = dict(M=m, N=n, ldx=ldx, ldy=ldy)
        if x_b & y_b:
            assert forward(y=y, **kw) == -1 and 'overlaps' in last()
        if x_b & s_b:
            assert forward(stats=stats, **kw) == -1 and 'overlaps' in last()
        if y_b & g_b:
            assert forward(x=P << 8, y=y, gamma=gamma, **kw) == -1 and 'overlaps' in last()
        if s_b & g_b:
            assert forward(x=P << 8, y=P << 9, stats=stats, gamma=gamma, **kw) == -1 and 'overlaps' in last()
        met += bool(x_b & y_b) + bool(x_b & s_b) + bool(y_b & g_b) + bool(s_b & g_b)
    assert met > 2000
