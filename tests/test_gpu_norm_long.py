"""GPU checks of layer norm's gradients over rows of millions of values."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import ends_ref as R
from rew_amd import eager as E
from rew_amd import ops as O

U = R.U
EPS = float(np.float32(1e-5))


@pytest.mark.parametrize("rows,n", [(3, 2 ** 21 - 7), (3, 2 ** 21 + 33), (1, 2 ** 27 + 21)])
def test_gradients(gpu, rows, n):
    """Both sides of 2^16 workgroups of the parameters' gradients, and as many values as take
    2^32 threads there.  Rows of seven values over and over, so that every sum is known; compared
    at both ends and in the middle."""
    r = np.random.default_rng(n)
    i = np.arange(n, dtype=np.int32) % 7
    count = np.bincount(i, minlength=7)
    xs, ds = r.integers(-8, 9, (rows, 7)) / 4.0, r.integers(-8, 9, (rows, 7)) / 8.0
    gs = 1.0 + r.integers(-4, 5, 7) / 16.0
    up = lambda a: E.fromHost(a.astype(np.float32)[..., i])  # noqa: E731
    x, dy, gamma = up(xs), up(ds), up(gs)
    beta = O.mul(gamma, O.broadcastTo(O.scalarF32(0.5), [n], []))
    y, stats = O.layerNorm(x, gamma, beta, withStats=True)
    mean = (xs * count).sum(1, keepdims=True) / n
    var = ((xs - mean) ** 2 * count).sum(1, keepdims=True) / n
    rstd = 1 / np.sqrt(var + EPS)
    h = (xs - mean) * rstd
    # (a chain of n / 1024 additions and some; its error in mean, variance and the two sums)
    c = (n / 1024 + 60) * U
    size = (np.abs(xs) * count).sum(1, keepdims=True) / n
    e_h = rstd * (2 * U * size + 2 * c * c * size + 3 * U * np.abs(xs)) + np.abs(h) * (c + 8 * U)
    grads = O.layerNormGrad(x, gamma, stats, dy)
    w = ds * gs
    m0, m1 = ((v * count).sum(1, keepdims=True) / n for v in (w, w * h))
    a0, a1 = ((v * count).sum(1, keepdims=True) / n for v in (np.abs(w), np.abs(w) * np.abs(h)))
    dx = rstd * (w - m0 - h * m1)
    e_dx = rstd * (6 * U * np.abs(w) + 2 * c * a0 + np.abs(h) * (2 * c * a1 + a0 * e_h.max()) +
                   e_h * np.abs(m1)) + (c + 12 * U) * np.abs(dx)
    dg, db = (ds * h).sum(0), ds.sum(0)
    e_dg = (np.abs(ds) * (e_h + 8 * U * np.abs(h))).sum(0) + 2 * U * np.abs(dg)
    e_y = np.abs(gs) * e_h + 4 * U * (np.abs(gs * h) + gs)
    for at in (0, n // 2, n - 40):
        k, cols = i[at:at + 40], ([at], [at + 40])
        rowwise = ([0, at], [rows, at + 40])
        R.check(O.slice_(y, *rowwise), (gs * h + 0.5 * gs)[:, k], e_y[:, k])
        R.check(O.slice_(grads[0], *rowwise), dx[:, k], e_dx[:, k])
        R.check(O.slice_(grads[1], *cols), dg[k], e_dg[k])
        R.check(O.slice_(grads[2], *cols), db[k], 0.0)  # (exact: multiples of 1 / 8)
