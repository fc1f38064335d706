"""GPU checks of infinities and NaN in gradOut: dV_j = sum_i P_ij gradOut_i has them in their
own columns, for the keys that their rows see, and nowhere else."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from test_gpu_packed import DTYPES, ints, make, tensor
from test_gpu_packed_special import SPECIAL


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 64), (6, 2, 128), (4, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", SPECIAL)
@pytest.mark.parametrize("at", [0, 45, 131, 159, 200])
@pytest.mark.parametrize("scale", [0.0, 4.0])
def test_grad_v(gpu, dtype, H, Hkv, D, causal, value, at, scale):
    """Scale 4: probabilities below the least of the operands' dtype, still above 0."""
    a, n, T = 70, 201, 301
    starts = [0, a, a + n, T]
    r = np.random.default_rng(D + at)
    (q, qh), (k, kh), (v, vh) = make(r, T, H, Hkv, D, dtype)
    do = tensor(r.standard_normal((T, H, D)), dtype)[1]
    cols = np.arange(3, D, 7)
    clean = do.copy()
    clean[a + at, :, cols] = 0.0
    do[a + at, :, cols] = value
    s = scale or D ** -0.5
    want, bnd = (x[2] for x in R.packed_grad(qh, kh, vh, starts, clean, causal, s, dtype))
    # float32 scores: 128 products lose at most 128 * 2^-24 of sum |q||k| s (below 2000 here at
    # the scale of 4: 1.6e-2 of a probability)
    slack = 1.6e-2 if scale else 0.0
    if slack:
        g, p = H // Hkv, np.zeros(want.shape)
        for b, e in zip(starts[:-1], starts[1:]):
            pr = R.attend(qh[b:e], kh[b:e], vh[b:e], 0, causal, s)[2]
            m = np.matmul(pr.transpose(0, 2, 1), np.abs(clean[b:e]).transpose(1, 0, 2))
            p[b:e] = m.reshape(Hkv, g, e - b, D).sum(1).transpose(1, 0, 2)
        bnd = bnd + slack * p
    out, stats = O.packedAttention(q, k, v, ints(starts), causal=causal, scale=scale, withLse=True)
    got = E.toHostF32(O.packedAttentionGrad(q, k, v, ints(starts), out, stats,
                                            tensor(do, dtype)[0], causal=causal,
                                            scale=scale)[2]).astype(np.float64)
    hit = np.zeros(got.shape, bool)
    seen = slice(a, a + at + 1 if causal else a + n)
    hit[seen, :, 3::7] = True
    np.testing.assert_array_equal(got[hit], np.full(hit.sum(), value))
    assert np.isfinite(got[~hit]).all()
    assert (np.abs(got - want)[~hit] <= bnd[~hit]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_opposite_infinities(gpu, dtype, causal):
    """Two rows' infinities of either sign in one column: NaN for keys that see both."""
    T, D = 300, 64
    r = np.random.default_rng(0)
    (q, _), (k, _), (v, _) = make(r, T, 4, 2, D, dtype)
    do = r.standard_normal((T, 4, D))
    do[100, :, 5], do[250, :, 5], do[280, :, 9] = np.inf, -np.inf, -np.inf
    out, stats = O.packedAttention(q, k, v, ints([0, T]), causal=causal, withLse=True)
    dv = E.toHostF32(O.packedAttentionGrad(q, k, v, ints([0, T]), out, stats,
                                           tensor(do, dtype)[0], causal=causal)[2])
    both = slice(0, 101 if causal else T)
    assert np.isnan(dv[both, :, 5]).all()
    if causal:
        assert (dv[101:251, :, 5] == -np.inf).all() and np.isfinite(dv[251:, :, 5]).all()
        assert np.isfinite(dv[281:]).all()
    assert (dv[:281 if causal else T, :, 9] == -np.inf).all()
    assert np.isfinite(np.delete(dv, [5, 9], axis=2)).all()
