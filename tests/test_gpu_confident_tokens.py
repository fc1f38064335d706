"""GPU checks of the loss of tokens whose target's logit stands far above the others, or lies
among large ones: the difference of two large numbers that is formed before either is rounded."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import ends_ref as R
from ends_ref import ints, tensor
from rew_amd import ops as O

U = R.U


def case(r, T, V, top, gap, dtype):
    """Logits top + d[v], exact in every form of the product: x = (top, 1), w = (1, d) with d a
    multiple of 1 / 4, 0 at word V // 2 and from -gap down at the others."""
    c = tensor(np.full(T, float(top)), dtype)[1]
    d = -gap - r.integers(0, 40, V) / 4.0
    d[V // 2] = 0.0
    x, xh = tensor(np.stack([c, np.ones(T)], 1), dtype)
    w, wh = tensor(np.stack([np.ones(V), d]), dtype)
    assert (xh[:, 0] == c).all() and (wh[1] == d).all()
    return x, w, xh, wh


def loss_and_bound(xh, wh, t):
    """The loss in float64 and its bound.  With exact logits: a rounding (U) for each addition
    of a value to a sum of exponentials near 1 (at most V of them, or V / 8 + 80 in the longest
    chain), what each word's exponential and its rescaling lose (its argument's rounding, the
    step of exp2, three joins), the logarithm and the two last operations."""
    z = xh @ wh
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    s = e.sum(1, keepdims=True)
    p, V = e / s, z.shape[1]
    at = (np.arange(len(t)), t)
    loss = np.log(s[:, 0]) + (m[:, 0] - z[at])
    lost = (p * np.where(z == m, 4.0, 4.0 * (m - z) + 24.0)).sum(1)
    return loss, U * (min(V, V / 8 + 80) + lost + 4 * np.abs(loss) + 8)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("T,V", [(1, 1), (5, 1), (3, 2), (70, 16), (300, 300), (600, 6000),
                                 (130, 33000)])
def test_target_on_top(gpu, dtype, T, V):
    r = np.random.default_rng(V)
    for top in (0.25, 20.0, -20.0, 61.0, 300.0, -310.0, 4000.0):
        for gap in (0.25, 8.0, 16.0):
            x, w, xh, wh = case(r, T, V, top, gap, dtype)
            t = np.full(T, V // 2)
            t[1::3] = r.integers(0, V, len(t[1::3]))  # and some words among the others
            want, bound = loss_and_bound(xh, wh, t)
            loss = O.linearCrossEntropy(x, w, ints(t))
            R.check(loss, want, bound)
            assert (R.host(loss) >= 0).all()


def test_one_word(gpu):
    """A vocabulary of one word: nothing to lose, whatever its logit."""
    r = np.random.default_rng(1)
    for H in (1, 40, 64, 200):
        x, _ = tensor(r.standard_normal((50, H)) * 20, "bfloat16")
        w, _ = tensor(r.standard_normal((H, 1)) * 20, "bfloat16")
        got = R.host(O.linearCrossEntropy(x, w, ints(np.zeros(50))))
        assert (got >= 0).all() and got.max() <= 13 * U, got.max()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("T,V", [(24, 16), (32, 300)])
def test_gradients_lose_one_rounding_of_lse(gpu, dtype, T, V):
    """lse is its value rounded once, and the probabilities are off by what that rounding is of
    them: gradX's first component, the sum of dz over the words, is next to 0."""
    r = np.random.default_rng(V)
    g = np.ones(T)
    h = R.HALF[dtype]
    for size in (8.0, 60.0, 300.0, 2000.0):
        for gap in (1.0, 8.0, 16.0):
            x, w, xh, wh = case(r, T, V, 0.0, gap, dtype)
            x, xh = tensor(np.stack([size * r.uniform(0.5, 1.0, T), np.ones(T)], 1), dtype)
            t = np.full(T, V // 2)
            lse, grad = O.linearCrossEntropy(x, w, ints(t), withLse=True)[1], tensor(g, "float32")[0]
            z = xh @ wh
            loss, e_loss = loss_and_bound(xh, wh, t)
            want = loss + z[np.arange(T), t]
            e_lse = U * np.abs(want) + e_loss
            R.check(lse, want, e_lse)
            dx, dw = O.linearCrossEntropyGrad(x, w, ints(t), lse, grad)
            d = z - want[:, None]
            dz = np.exp(d)
            e_dz = dz * (e_lse[:, None] + (4 * np.abs(d) + 8) * U) + U
            dz[np.arange(T), t] = np.expm1(-loss)
            e_dz += (h * h + 6 * U) * np.abs(dz) + (2.0 ** -39 if dtype == "float16" else 0.0)
            for got, a, b in ((dx, dz, wh.T), (dw, xh.T, dz)):
                want = a @ b
                off = np.abs(a) @ e_dz if b is dz else e_dz @ np.abs(b)
                off += 2 * (max(T, V) + 8) * U * (np.abs(a) @ np.abs(b))
                R.check(got, want, off + (h + 4 * U) * np.abs(want) + R.TINY[dtype])
