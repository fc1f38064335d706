"""GPU checks of scores of -infinity: such a key weighs nothing, and a row that has no other gives
zeros, as one that sees no key."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from rew_amd import eager as E
from rew_amd import ops as O
from test_gpu_packed import DTYPES, ints, tensor


def rows(n, D):
    """q of ones; k of zeros with -infinity in the first column of the first `n` tokens; v of the
    tokens' numbers."""
    T = n + 3
    q, k, v = np.ones((T, 2, D)), np.zeros((T, 1, D)), np.zeros((T, 1, D))
    k[:n, :, 0] = -np.inf
    v[:] = np.arange(T)[:, None, None] % 7
    want = np.zeros((T, 2, D))
    for t in range(n, T):
        want[t] = v[n:t + 1].mean(0)
    return q, k, v, want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("n", [1, 40, 130])
def test_packed(gpu, dtype, D, n):
    q, k, v, want = rows(n, D)
    out, stats = O.packedAttention(*(tensor(x, dtype)[0] for x in (q, k, v)), ints([0, n + 3]),
                                   withLse=True)
    np.testing.assert_allclose(E.toHostF32(out), want, rtol=2 ** -7)
    lse = E.toHost(stats.lse)
    assert np.isneginf(lse[:n]).all() and np.isfinite(lse[n:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width", [(1, 20), (40, 20), (40, 400), (1500, 100), (1500, 400)])
@pytest.mark.parametrize("new", [4, 140])
def test_paged(gpu, dtype, n, width, new):
    D, page = 64, 16
    q, k, v, want = rows(n, D)
    T = len(q)
    new = min(new, T)
    kp, vp = (E.empty(DTYPES[dtype], (-(-T // page), 1, page, D)) for _ in range(2))
    O.pagedCacheWrite(kp, vp, tensor(k, dtype)[0], tensor(v, dtype)[0], ints(np.arange(T)))
    table = np.full((1, width), -1)
    table[0, :kp.shape[0]] = np.arange(kp.shape[0])
    out = O.pagedAttention(tensor(q[T - new:], dtype)[0], kp, vp, ints(table), ints([0, new]),
                           ints([T]), maxNew=new)
    np.testing.assert_allclose(E.toHostF32(out), want[T - new:], rtol=2 ** -7)
