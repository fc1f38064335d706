"""GPU checks of results below float16's normal range (2^-14), where a rounding takes up to 2^-25
whatever the value: the rest that the forward pass leaves, and the gradient of q through it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from test_gpu_packed import DTYPES, ints, make, tensor

LEAST = {"float16": 2.0 ** -14, "bfloat16": 2.0 ** -100}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("size", [2.0 ** -23, 2.0 ** -18, 2.0 ** -15, 2.0 ** -12])
def test_small_values(gpu, dtype, D, size):
    starts, h = [0, 90, 200], R.HALF[dtype]
    r = np.random.default_rng(D)
    (q, qh), (k, kh), (v, vh) = make(r, 200, 4, 2, D, dtype)
    v, vh = tensor(vh * size, dtype)
    do, doh = tensor(r.standard_normal(qh.shape) * 2 ** 9, dtype)
    out, stats = O.packedAttention(q, k, v, ints(starts), withLse=True)
    want, _, mag = R.packed(qh, kh, vh, starts, True, D ** -0.5)
    got = E.toHostF32(out).astype(np.float64)
    most = np.maximum(np.abs(got).max(2, keepdims=True), LEAST[dtype])
    rest = E.toHost(stats.rest)
    # out with its rest: a rounding of the probabilities, float32, a step of the rest
    step = most * h / 127
    assert (np.abs(got + rest * step - want) <= (h + R.F32) * mag + step).all()
    # dQ: packed_grad counts half a step of the rest of each row's own largest; here at least of
    # LEAST, times sum |gradOut|, sum p = 1 and max |k|
    g = O.packedAttentionGrad(q, k, v, ints(starts), out, stats, do)[0]
    wants, bnds = R.packed_grad(qh, kh, vh, starts, doh, True, D ** -0.5, dtype)
    slack = 1.1 * h / 254 * LEAST[dtype] * np.abs(doh).sum(2, keepdims=True) * np.abs(kh).max()
    over = np.abs(E.toHostF32(g) - wants[0]) - bnds[0] - slack * D ** -0.5 - 2.0 ** -25
    assert over.max() <= 0, over.max()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_zeros(gpu, dtype):
    """V of zeros: out and rest are zeros, and the gradients of q and k too."""
    (q, _), (k, _), _ = make(np.random.default_rng(0), 70, 4, 2, 64, dtype)
    v = tensor(np.zeros((70, 2, 64)), dtype)[0]
    out, stats = O.packedAttention(q, k, v, ints([0, 70]), withLse=True)
    assert not E.toHostF32(out).any() and not E.toHost(stats.rest).any()
    dq, dk, dv = O.packedAttentionGrad(q, k, v, ints([0, 70]), out, stats, q)
    assert not E.toHostF32(dq).any() and not E.toHostF32(dk).any() and E.toHostF32(dv).any()
