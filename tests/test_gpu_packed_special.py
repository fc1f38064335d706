"""GPU checks of infinities and NaN in places that a row does not see: keys of later tokens,
other sequences, rows of no sequence, and the gradients' shared scale."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from test_gpu_packed import DTYPES, check, ints, make, tensor
from test_gpu_paged import paged_call, paged_case, paged_want

SPECIAL = [np.nan, np.inf, -np.inf]


def put(h, rows, value, dtype):
    """h with `value` in some places of the given rows; (tensor, values)."""
    h = h.copy()
    for i, row in enumerate(rows):
        h[row, :, (3 + 5 * i) % h.shape[2]:: 7] = value
    return tensor(h, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 64), (6, 2, 128)])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("value", SPECIAL)
def test_packed_later_keys(gpu, dtype, H, Hkv, D, which, value):
    """Rows before the token that holds it, and other sequences, have the results that they
    have without it; the rows that see it in V get it."""
    starts, at = [0, 100, 330, 335, 400], 100 + 45
    r = np.random.default_rng(D)
    (q, _), (k, kh), (v, vh) = make(r, 420, H, Hkv, D, dtype)
    clean = E.toHostF32(O.packedAttention(q, k, v, ints(starts)))
    bad, badh = put(kh if which == "k" else vh, [at, at + 130], value, dtype)
    args = (q, bad, v) if which == "k" else (q, k, bad)
    got = E.toHostF32(O.packedAttention(*args, ints(starts)))
    safe = np.r_[0:at, 330:420]
    if which == "k":  # (the max of a wave's other rows may have moved: an ulp)
        h = R.HALF[dtype]
        np.testing.assert_allclose(got[safe], clean[safe], rtol=4 * h, atol=4 * h)
        assert np.isfinite(got[safe]).all()
    else:
        np.testing.assert_array_equal(got[safe], clean[safe])
        g = H // Hkv
        seen = np.repeat(badh[at], g, axis=0)
        for row in (at, at + 1, at + 100):
            np.testing.assert_array_equal(got[row][~np.isfinite(seen)],
                                          seen[~np.isfinite(seen)])
            if row < at + 130:
                np.testing.assert_array_equal(got[row][np.isfinite(seen)],
                                              clean[row][np.isfinite(seen)])


@pytest.mark.parametrize("news,lens,width", [
    ([3, 1, 6], [130, 40, 6], None), ([3, 1, 6], [130, 40, 6], 300),
    ([150, 1, 70], [500, 300, 70], None)], ids=["few", "few_wide", "chunks"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("value", SPECIAL)
def test_paged_later_keys(gpu, news, lens, width, dtype, D, value):
    """The last new token of each request holds it in V: only its own row sees it."""
    r = np.random.default_rng(D + len(news))
    c = paged_case(r, news, lens, 8, 2, D, 16, dtype, width=width)
    clean = E.toHostF32(paged_call(c))
    for n, row in zip(lens, c["table"]):
        c["vh"][row[(n - 1) // 16], :, (n - 1) % 16, 3::7] = value
    flat = c["vh"].transpose(0, 2, 1, 3).reshape(-1, 2, D)
    k = c["kh"].transpose(0, 2, 1, 3).reshape(-1, 2, D)
    O.pagedCacheWrite(c["kp"], c["vp"], tensor(k, dtype)[0], tensor(flat, dtype)[0],
                      ints(np.arange(len(flat))))
    got = E.toHostF32(paged_call(c))
    last = np.cumsum(news) - 1
    rest = np.setdiff1d(np.arange(sum(news)), last)
    np.testing.assert_array_equal(got[rest], clean[rest])
    np.testing.assert_array_equal(got[last][..., 3::7], np.full(got[last][..., 3::7].shape, value))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("value", SPECIAL + [3e4])
@pytest.mark.parametrize("which", range(4), ids=["q", "k", "v", "do"])
def test_grad_of_other_sequences(gpu, dtype, causal, value, which):
    """A sequence's gradients do not depend on what another one, or the rows of none, hold
    (a large finite value in another sequence may: float16's shared scale)."""
    starts = [0, 70, 230, 301]
    H, Hkv, D, T = 6, 2, 64, 320
    r = np.random.default_rng(int(causal))
    x = [h for _, h in make(r, T, H, Hkv, D, dtype)] + [r.standard_normal((T, H, D)) * 1e-3]
    x[3] = tensor(x[3], dtype)[1]
    want, bnd = R.packed_grad(*x[:3], starts, x[3], causal, D ** -0.5, dtype)
    rows = [301, 319] + ([] if np.isfinite(value) else [75, 140, 229])
    x[which] = put(x[which], rows, value, dtype)[1]
    q, k, v, do = (tensor(y, dtype)[0] for y in x)
    out, stats = O.packedAttention(q, k, v, ints(starts), causal=causal, withLse=True)
    got = O.packedAttentionGrad(q, k, v, ints(starts), out, stats, do, causal=causal)
    for g, w, b in zip(got, want, bnd):
        g = E.toHostF32(g).astype(np.float64)
        for rows in (slice(0, 70), slice(230, 301)):
            assert np.isfinite(g[rows]).all()
            assert (np.abs(g[rows] - w[rows]) <= b[rows]).all()
        assert (g[301:] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 64), (6, 2, 128), (4, 1, 128)])
@pytest.mark.parametrize("value", SPECIAL)
@pytest.mark.parametrize("which", range(4), ids=["q", "k", "v", "do"])
@pytest.mark.parametrize("at", [0, 45, 131, 159])
def test_causal_grad_of_one_token(gpu, dtype, H, Hkv, D, value, which, at):
    """A token's infinities or NaN in k or v do not reach the gradient of q of rows before it,
    those in q or gradOut only its own row's and not the keys behind it."""
    a, n, T = 70, 160, 301
    starts = [0, a, a + n, T]
    r = np.random.default_rng(D + which)
    x = [h for _, h in make(r, T, H, Hkv, D, dtype)] + [r.standard_normal((T, H, D))]
    x[3] = tensor(x[3], dtype)[1]
    want, bnd = R.packed_grad(*x[:3], starts, x[3], True, D ** -0.5, dtype)
    x[which] = put(x[which], [a + at], value, dtype)[1]
    q, k, v, do = (tensor(y, dtype)[0] for y in x)
    out, stats = O.packedAttention(q, k, v, ints(starts), withLse=True)
    got = [E.toHostF32(g).astype(np.float64)
           for g in O.packedAttentionGrad(q, k, v, ints(starts), out, stats, do)]
    own, rows = np.arange(a + at, a + at + 1), np.arange(T)
    later = np.r_[a + at:a + n]
    if which in (1, 2):  # k, v: rows that see it; every key has such a row behind it
        clean = [np.setdiff1d(rows, later), np.r_[0:a, a + n:T], np.r_[0:a, a + n:T]]
    else:
        clean = [np.setdiff1d(rows, own)] + [np.r_[0:a, a + at + 1:T]] * 2
    for g, w, b, c in zip(got, want, bnd, clean):
        assert np.isfinite(g[c]).all()
        assert (np.abs(g[c] - w[c]) <= b[c]).all()
    assert not np.isfinite(got[0][own]).all() and not np.isfinite(got[1][a:a + at + 1]).all()
