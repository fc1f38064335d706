"""GPU checks of ``ops.linearCrossEntropy`` and its gradients against float64."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import ends_ref as R
from ends_ref import ints, tensor
from rew_amd import ops as O
from rew_amd.eager import DType
from rew_amd import eager as E

DTYPES = ["bfloat16", "float16"]


def f32(a):
    return E.fromHost(np.asarray(a, np.float32), DType.FLOAT32)


def case(r, T, H, V, dtype, tied, std=2.0):
    x, xh = tensor(r.standard_normal((T, H)), dtype)
    w, wh = tensor(r.standard_normal((V, H) if tied else (H, V)) * std / H ** 0.5, dtype)
    targets = np.where(r.random(T) < 0.1, -1, r.integers(0, V, T))
    grad = r.uniform(0.5, 1.5, T).astype(np.float32)
    return (x, w, ints(targets), f32(grad)), (xh, wh.T if tied else wh, targets,
                                              grad.astype(np.float64))


def run(t, h, dtype, tied):
    (x, w, targets, grad), (xh, wh, th, gh) = t, h
    loss, lse = O.linearCrossEntropy(x, w, targets, tied, withLse=True)
    for got, (want, bound) in zip((loss, lse), R.cross_entropy(xh, wh, th)):
        R.check(got, want, bound)
    np.testing.assert_array_equal(R.host(loss), R.host(O.linearCrossEntropy(x, w, targets, tied)))
    got = O.linearCrossEntropyGrad(x, w, targets, lse, grad, tied)
    (dx, e_dx), (dw, e_dw) = R.cross_entropy_grad(xh, wh, th, gh, dtype)
    R.check(got[0], dx, e_dx)
    R.check(got[1], dw.T if tied else dw, e_dw.T if tied else e_dw)
    for a, c in zip(got, O.linearCrossEntropyGrad(x, w, targets, lse, grad, tied)):
        np.testing.assert_array_equal(R.host(a), R.host(c))  # the same call, the same bits


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,V", [
    (1, 1, 1), (1, 64, 2), (3, 8, 8), (5, 7, 9), (64, 64, 256), (65, 72, 264), (100, 256, 1000),
    (255, 63, 257), (257, 130, 511), (256, 128, 512), (300, 65, 1025), (2, 1000, 40),
    (513, 320, 700)])
def test_sizes(gpu, tied, dtype, T, H, V):
    run(*case(np.random.default_rng(T + V), T, H, V, dtype, tied), dtype, tied)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,V", [
    (1, 1, 2), (1, 64, 2), (2, 64, 2), (5, 3, 1000), (31, 64, 300), (32, 1, 300), (32, 72, 40),
    (7, 1000, 5000), (16, 200, 60001), (32, 128, 40000)])
def test_few_tokens(gpu, tied, dtype, T, H, V):
    """Gradients that are sums of few terms: rounded once, as dz keeps its remainder."""
    (x, w, targets, grad), (xh, wh, th, gh) = case(np.random.default_rng(T * V), T, H, V, dtype,
                                                   tied)
    lse = O.linearCrossEntropy(x, w, targets, tied, withLse=True)[1]
    got = O.linearCrossEntropyGrad(x, w, targets, lse, grad, tied)
    (dx, e_dx), (dw, e_dw) = R.cross_entropy_grad(xh, wh, th, gh, dtype, rest=True)
    R.check(got[0], dx, e_dx)
    R.check(got[1], dw.T if tied else dw, e_dw.T if tied else e_dw)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("V", [33000, 33001])
def test_pieces_of_the_vocabulary(gpu, tied, V):
    """More columns than are held at a time, aligned and not."""
    run(*case(np.random.default_rng(V), 2100, 40, V, "bfloat16", tied), "bfloat16", tied)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_targets_and_no_tokens(gpu, tied, dtype):
    r = np.random.default_rng(1)
    (x, w, _, grad), (xh, wh, _, _) = case(r, 20, 48, 100, dtype, tied)
    for t in ([-1] * 20, [100] * 20, [-2 ** 31] * 20, [2 ** 31 - 1] * 20):
        loss, lse = O.linearCrossEntropy(x, w, ints(t), tied, withLse=True)
        R.check(loss, np.zeros(20), 0.0)
        R.check(lse, *R.cross_entropy(xh, wh, t)[1])
        for g, like in zip(O.linearCrossEntropyGrad(x, w, ints(t), lse, grad, tied), (x, w)):
            R.check(g, np.zeros(like.shape), 0.0)
    none = tensor(np.zeros((0, 48)), dtype)[0]
    loss, lse = O.linearCrossEntropy(none, w, ints([]), tied, withLse=True)
    assert loss.shape == (0,)
    dx, dw = O.linearCrossEntropyGrad(none, w, ints([]), lse, f32([]), tied)
    assert dx.shape == (0, 48)
    R.check(dw, np.zeros(w.shape), 0.0)


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("H", [64, 50])
def test_padding_may_hold_anything(gpu, tied, H):
    """x and gradLoss of tokens without a target, infinities and NaN included, reach nothing."""
    r = np.random.default_rng(H)
    (x, w, _, _), (xh, wh, th, gh) = case(r, 70, H, 300, "bfloat16", tied)
    bad, bad_g = xh.copy(), gh.copy()
    for i, v in ((3, np.nan), (9, np.inf), (40, -np.inf), (69, np.nan)):
        th[i], bad[i], bad_g[i] = -1, v, v
    t = ints(th)
    out = []
    for xv, gv in ((np.where(th[:, None] < 0, 0.0, xh), np.where(th < 0, 0.0, gh)), (bad, bad_g)):
        xt = tensor(xv, "bfloat16")[0]
        loss, lse = O.linearCrossEntropy(xt, w, t, tied, withLse=True)
        out.append([R.host(loss)] + [R.host(g) for g in O.linearCrossEntropyGrad(
            xt, w, t, lse, f32(gv), tied)])
    for a, c in zip(*out):
        np.testing.assert_array_equal(a, c)


def test_infinities_stay_in_their_rows(gpu):
    r = np.random.default_rng(2)
    (x, w, t, grad), (xh, wh, th, gh) = case(r, 300, 64, 500, "bfloat16", False)
    bad = xh.copy()
    bad[5, 3], bad[299, 0] = np.nan, np.inf
    th[[5, 299]] = 1
    t = ints(th)
    keep = np.setdiff1d(np.arange(300), [5, 299])
    want, lse0 = O.linearCrossEntropy(x, w, t, withLse=True)
    xt = tensor(bad, "bfloat16")[0]
    loss, lse = O.linearCrossEntropy(xt, w, t, withLse=True)
    np.testing.assert_array_equal(R.host(loss)[keep], R.host(want)[keep])
    assert not np.isfinite(R.host(loss)[[5, 299]]).any()
    dx = R.host(O.linearCrossEntropyGrad(xt, w, t, lse, grad)[0])
    np.testing.assert_array_equal(dx[keep],
                                  R.host(O.linearCrossEntropyGrad(x, w, t, lse0, grad)[0])[keep])


def test_infinite_logits(gpu):
    """One logit of +infinity: lse is infinite, the loss 0/0 at it and infinite elsewhere; all
    -infinity: lse -infinity; some -infinity: no part."""
    w = np.ones((1, 8))
    x = np.array([[1.0], [-1.0]])
    w[0, 3] = np.inf
    wt = tensor(w, "float16")[0]
    loss, lse = (R.host(v) for v in O.linearCrossEntropy(tensor(x, "float16")[0], wt,
                                                         ints([0, 0]), withLse=True))
    assert lse[0] == np.inf and loss[0] == np.inf
    assert abs(lse[1] - (-1 + np.log(7))) < 1e-6 and abs(loss[1] - np.log(7)) < 1e-6
    w[0, :] = np.inf
    lse = R.host(O.linearCrossEntropy(tensor([[-1.0]], "float16")[0], tensor(w, "float16")[0],
                                      ints([-1]), withLse=True)[1])
    assert lse[0] == -np.inf


@pytest.mark.parametrize("tied", [True, False])
@pytest.mark.parametrize("H", [8, 72, 100, 320])
@pytest.mark.parametrize("T,V", [(3, 56), (700, 6000)])
def test_infinite_weights(gpu, tied, H, T, V):
    """A word whose logit is -infinity takes no part, whatever the width of the rows; one of
    +infinity makes lse infinite.  The logits of the others are zero: log(V - 1), to a few
    roundings of a float32 sum of ones (exact) and its logarithm."""
    w = np.zeros((V, H))
    w[5] = -np.inf
    x = tensor(np.ones((T, H)), "bfloat16")[0]
    t = ints(np.arange(T) % 4)
    wt = tensor(w if tied else w.T, "bfloat16")[0]
    loss, lse = O.linearCrossEntropy(x, wt, t, tied=tied, withLse=True)
    np.testing.assert_allclose(R.host(loss), np.log(V - 1), rtol=4 * 2.0 ** -24)
    dw = R.host(O.linearCrossEntropyGrad(x, wt, t, lse, f32(np.ones(T)), tied=tied)[1])
    dw = dw if tied else dw.T
    assert np.isfinite(dw).all() and not dw[5].any()
    w[5, 0] = np.inf
    w[5, 1:] = 0.0
    lse = O.linearCrossEntropy(x, tensor(w if tied else w.T, "bfloat16")[0], t, tied=tied,
                               withLse=True)[1]
    assert (R.host(lse) == np.inf).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 1e20])
def test_size_of_the_gradient(gpu, dtype, size):
    """gradLoss of any size, spread over several powers of two and zero: dx of bfloat16 keeps
    its relative error; float16's results are compared where they do not overflow."""
    if dtype == "float16" and size > 1e4:
        pytest.skip("float16 results overflow")
    r = np.random.default_rng(3)
    (x, w, t, _), (xh, wh, th, gh) = case(r, 130, 96, 400, dtype, False)
    g = (gh * size * 2.0 ** -r.integers(0, 12, 130)).astype(np.float32)
    g[7] = 0.0
    lse = O.linearCrossEntropy(x, w, t, withLse=True)[1]
    for got, (want, bound) in zip(O.linearCrossEntropyGrad(x, w, t, lse, f32(g)),
                                  R.cross_entropy_grad(xh, wh, th, g.astype(np.float64), dtype)):
        R.check(got, want, bound)
    zero = O.linearCrossEntropyGrad(x, w, t, lse, f32(np.zeros(130)))
    for got in zero:
        assert not R.host(got).any()


def test_peaked_and_large_logits(gpu):
    """Logits of some hundreds: probabilities of one and of zero."""
    r = np.random.default_rng(8)
    for dtype in DTYPES:
        run(*case(r, 90, 128, 600, dtype, True, std=60.0), dtype, True)


def test_gradient_against_differences(gpu):
    """Central differences of the float64 loss, at the kernel's own (rounded) x and weight."""
    r = np.random.default_rng(9)
    (x, w, t, grad), (xh, wh, th, gh) = case(r, 12, 16, 40, "bfloat16", False)
    lse = O.linearCrossEntropy(x, w, t, withLse=True)[1]
    dx, dw = O.linearCrossEntropyGrad(x, w, t, lse, grad)
    (wx, bx), (ww, bw) = R.cross_entropy_grad(xh, wh, th, gh, "bfloat16")

    def f(xv, wv):
        return (gh * R.cross_entropy(xv, wv, th)[0][0]).sum()

    for k, (v, d, b) in enumerate(((xh, R.host(dx), bx), (wh, R.host(dw), bw))):
        for i in r.choice(v.size, 20, replace=False):
            at = np.unravel_index(i, v.shape)
            side = []
            for s in (1e-4, -1e-4):
                args = [xh.copy(), wh.copy()]
                args[k][at] += s
                side.append(f(*args))
            assert abs((side[0] - side[1]) / 2e-4 - d[at]) <= b[at] + 1e-7
