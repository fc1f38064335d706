"""GPU checks of the cross entropy of very many tokens: beyond 2^17, and 2^30, which the library
itself refuses."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import ends_ref as R
from ends_ref import host, ints, tensor
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType, EagerError


def test_library_refusals(gpu):
    T = 2 ** 30
    x, w, t = (E.empty(DType.BFLOAT16, (T, 1)), E.empty(DType.BFLOAT16, (1, 7)),
               E.empty(DType.INT32, (T,)))
    f = E.empty(DType.FLOAT32, (T,))
    for op, ins, attrs in (("linearCrossEntropy", [x, w, t], [("stats", "true")]),
                           ("linearCrossEntropyGrad", [x, w, t, f, f], [])):
        with pytest.raises(EagerError, match="2\\^30 tokens"):
            E.dispatchEager(op, ins, [("tied", "false"), *attrs])


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("T,H,V", [(2 ** 17 + 5000, 64, 16500), (2 ** 20 + 7, 8, 4500)])
def test_pieces_get_smaller(gpu, tied, T, H, V):
    """Beyond 2^17 tokens fewer words are held at a time: the loss, the gradients of some tokens
    (every word) and of some words (every token), those on both sides of a piece's end among
    them."""
    r = np.random.default_rng(T)
    piece = -(-(2 ** 31 // T) // 256) * 256
    assert V > piece
    x, xh = tensor(1.0 + 0.5 * r.standard_normal((T, H)), "bfloat16")
    w, wh = tensor(r.standard_normal((V, H) if tied else (H, V)) * 2 / H ** 0.5, "bfloat16")
    wh = wh.T if tied else wh
    # (targets of half the tokens, so that their sums do not cancel)
    words = np.array([0, 1, piece - 1, piece, V - 1])
    t = np.where(r.random(T) < 0.5, r.choice(words, T), r.integers(-1, V, T))
    g = r.uniform(0.5, 1.5, T).astype(np.float32)
    loss, lse = O.linearCrossEntropy(x, w, ints(t), tied, withLse=True)
    dx, dw = O.linearCrossEntropyGrad(x, w, ints(t), lse, E.fromHost(g), tied)
    rows = np.concatenate([np.arange(6), T // 2 + np.arange(5), T - 1 - np.arange(6)])
    lse, gh = host(lse), g.astype(np.float64)
    for got, (want, bound) in zip((host(loss), lse), R.cross_entropy(xh[rows], wh, t[rows])):
        assert (np.abs(got[rows] - want) <= bound).all()
    (want, bound), _ = R.cross_entropy_grad(xh[rows], wh, t[rows], gh[rows], "bfloat16")
    assert (np.abs(host(dx)[rows] - want) <= bound).all()
    # dw of some words, given the (checked) lse: p's relative error from it and the logit
    live = t >= 0
    z = xh @ wh[:, words]
    e_z = 2 * (H + 4) * R.U * (np.abs(xh) @ np.abs(wh[:, words]))
    p = np.exp(z - lse[:, None])
    dz = np.where(live, gh, 0.0)[:, None] * (p - (t[:, None] == words))
    e_dz = np.where(live, gh, 0.0)[:, None] * (p * (np.expm1(e_z) + (
        4 * np.abs(z - lse[:, None]) + 2 * np.abs(lse[:, None]) + 8) * R.U) + R.U) + (
        R.HALF["bfloat16"] + 6 * R.U) * np.abs(dz)
    want = xh.T @ dz
    # (a product's instruction adds 16 terms to a sum)
    bound = np.abs(xh).T @ e_dz + 2 * (T / 16 + 64) * R.U * (np.abs(xh).T @ np.abs(dz))
    assert np.median(bound / np.abs(want)) < 0.02
    got = host(dw).T if tied else host(dw)
    assert (np.abs(got[:, words] - want) <= bound + R.HALF["bfloat16"] * np.abs(want)).all()
