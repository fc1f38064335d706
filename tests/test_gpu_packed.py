"""GPU checks of attention over packed sequences and its gradients, against float64 forms
(packed_ref) with bounds that count the kernels' roundings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType

DTYPES = {"bfloat16": DType.BFLOAT16, "float16": DType.FLOAT16}


def tensor(x, dtype):
    """(device tensor, its values in float64)."""
    t = E.fromHost(np.asarray(x, np.float32), DTYPES[dtype])
    return t, E.toHostF32(t).astype(np.float64)


def ints(x):
    return E.fromHost(np.asarray(x, np.int32))


def check(got, want, bound):
    got = E.toHostF32(got).astype(np.float64)
    assert got.shape == want.shape
    over = np.abs(got - want) - bound
    assert np.isfinite(got).all()
    assert over.max(initial=-1.0) <= 0.0, (over.max(), np.unravel_index(over.argmax(), over.shape))


def make(r, T, H, Hkv, D, dtype):
    return (tensor(r.standard_normal((T, H, D)) * 1.5, dtype),
            tensor(r.standard_normal((T, Hkv, D)), dtype),
            tensor(r.standard_normal((T, Hkv, D)), dtype))


LENGTHS = {
    "one": [1], "few": [5, 1, 3], "tile": [64], "past_tile": [65, 63], "tiles": [128, 129, 127],
    "ragged": [33, 300, 1, 0, 190, 77], "long": [700],
}


@pytest.mark.parametrize("lens", LENGTHS, ids=list(LENGTHS))
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 64), (4, 1, 128), (6, 2, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention(gpu, lens, H, Hkv, D, dtype, causal):
    lens = LENGTHS[lens]
    r = np.random.default_rng(sum(lens) + H + D)
    starts = np.concatenate([[0], np.cumsum(lens)])
    (q, qh), (k, kh), (v, vh) = make(r, starts[-1], H, Hkv, D, dtype)
    out, (lse, rest) = O.packedAttention(q, k, v, ints(starts), causal=causal, withLse=True)
    want, wl, mag = R.packed(qh, kh, vh, starts, causal, D ** -0.5)
    check(out, want, R.out_bound(want, mag, dtype))
    np.testing.assert_array_equal(
        E.toHost(out), E.toHost(O.packedAttention(q, k, v, ints(starts), causal=causal)))
    # out with its rest: half a step of the rest in place of the output's rounding
    got = E.toHostF32(out).astype(np.float64)
    step = np.abs(got).max(2, keepdims=True) * R.HALF[dtype] / 127
    # (a float16 below 2^-14 is rounded by more than 2^-11 of itself: 2^-25)
    got += E.toHost(rest) * step
    assert (np.abs(got - want) <= (R.HALF[dtype] + R.F32) * mag + step + 2.0 ** -25).all()
    # no rounding to the dtype in it: the scores' and the sum's float32
    check(lse, wl, R.F32 + 1e-6 * np.abs(wl))


def test_packed_rows_of_no_sequence_are_zero(gpu):
    r = np.random.default_rng(3)
    starts = np.array([7, 40, 40, 171])
    (q, qh), (k, kh), (v, vh) = make(r, 300, 4, 2, 64, "bfloat16")
    (g, gh) = tensor(r.standard_normal((300, 4, 64)), "bfloat16")
    out, stats = O.packedAttention(q, k, v, ints(starts), withLse=True)
    want, wl, mag = R.packed(qh, kh, vh, starts, True, 0.125)
    check(out, want, R.out_bound(want, mag, "bfloat16"))
    np.testing.assert_array_equal(np.isneginf(E.toHost(stats.lse)), np.isneginf(wl))
    res, bnd = R.packed_grad(qh, kh, vh, starts, gh, True, 0.125, "bfloat16")
    for t, w, b in zip(O.packedAttentionGrad(q, k, v, ints(starts), out, stats, g), res, bnd):
        check(t, w, b)
        assert not E.toHostF32(t)[:7].any() and not E.toHostF32(t)[171:].any()


@pytest.mark.parametrize("starts", [[0], [0, 0], [5, 5]])
def test_packed_without_tokens_in_sequences(gpu, starts):
    (q, _), (k, _), (v, _) = make(np.random.default_rng(1), 9, 2, 1, 32, "float16")
    out, stats = O.packedAttention(q, k, v, ints(starts), withLse=True)
    assert not E.toHostF32(out).any() and np.isneginf(E.toHost(stats.lse)).all()
    for t in O.packedAttentionGrad(q, k, v, ints(starts), out, stats, q):
        assert not E.toHostF32(t).any()


def test_packed_no_tokens(gpu):
    q = E.empty(DType.BFLOAT16, (0, 4, 64))
    k = E.empty(DType.BFLOAT16, (0, 2, 64))
    out, stats = O.packedAttention(q, k, k, ints([0]), withLse=True)
    assert out.shape == (0, 4, 64) and E.toHost(stats.lse).shape == (0, 4)
    dq, dk, dv = O.packedAttentionGrad(q, k, k, ints([0]), out, stats, q)
    assert E.toHost(dq).size == E.toHost(dk).size == E.toHost(dv).size == 0


def test_packed_starts_out_of_order_stay_inside(gpu):
    """Wrong starts give some result, and the sequences before the fault the right one."""
    r = np.random.default_rng(8)
    (q, qh), (k, kh), (v, vh) = make(r, 100, 2, 2, 64, "bfloat16")
    out, stats = O.packedAttention(q, k, v, ints([0, 60, 20, 5000, -3]), withLse=True)
    want, _, mag = R.packed(qh, kh, vh, np.array([0, 60]), True, 0.125)
    got = E.toHostF32(out)[:20]
    assert (np.abs(got - want[:20]) <= R.out_bound(want, mag, "bfloat16")[:20]).all()
    O.packedAttentionGrad(q, k, v, ints([0, 60, 20, 5000, -3]), out, stats, q)
    E.sync()


def test_packed_scale_and_large_scores(gpu):
    """A given scale; scores up to several hundred, where the running max must move."""
    r = np.random.default_rng(5)
    for dtype in DTYPES:
        (q, qh), (k, kh), (v, vh) = make(r, 200, 2, 1, 64, dtype)
        k, kh = tensor(kh * np.linspace(0.1, 8.0, 200)[:, None, None], dtype)
        out = O.packedAttention(q, k, v, ints([0, 200]), scale=0.5)
        # float32 scores: 64 * 2^-24 of sum |q||k| 0.5 (at most 1500 here) is 6e-3 of a probability
        want, _, mag = R.packed(qh, kh, vh, np.array([0, 200]), True, 0.5)
        check(out, want, R.out_bound(want, mag, dtype) + 6e-3 * mag)


GRADS = {"one": [1], "few": [5, 1, 3], "tile": [128], "ragged": [33, 300, 1, 0, 190], "long": [500]}


@pytest.mark.parametrize("lens", GRADS, ids=list(GRADS))
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 64), (4, 1, 128), (6, 2, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_grad(gpu, lens, H, Hkv, D, dtype, causal):
    lens = GRADS[lens]
    r = np.random.default_rng(sum(lens) + H + D + 1)
    starts = np.concatenate([[0], np.cumsum(lens)])
    (q, qh), (k, kh), (v, vh) = make(r, starts[-1], H, Hkv, D, dtype)
    (g, gh) = tensor(r.standard_normal((starts[-1], H, D)), dtype)
    s = ints(starts)
    out, stats = O.packedAttention(q, k, v, s, causal=causal, withLse=True)
    got = O.packedAttentionGrad(q, k, v, s, out, stats, g, causal=causal)
    res, bnd = R.packed_grad(qh, kh, vh, starts, gh, causal, D ** -0.5, dtype)
    for t, w, b in zip(got, res, bnd):
        check(t, w, b)


@pytest.mark.parametrize("size", [1e-4, 1.0, 3e3])
def test_packed_grad_float16_of_any_size(gpu, size):
    """float16 gradients from loss scales of many sizes: dS is stored scaled."""
    r = np.random.default_rng(11)
    starts = np.array([0, 150, 260])
    (q, qh), (k, kh), (v, vh) = make(r, 260, 4, 2, 64, "float16")
    (g, gh) = tensor(r.standard_normal((260, 4, 64)) * size, "float16")
    out, stats = O.packedAttention(q, k, v, ints(starts), withLse=True)
    res, bnd = R.packed_grad(qh, kh, vh, starts, gh, True, 0.125, "float16")
    for t, w, b in zip(O.packedAttentionGrad(q, k, v, ints(starts), out, stats, g), res, bnd):
        # a result below 2^-14 is rounded to a multiple of 2^-24
        check(t, w, b + 2.0 ** -25)


def test_packed_grad_against_differences(gpu):
    """The formulas' gradients against central differences of the float64 forward form."""
    r = np.random.default_rng(2)
    starts = np.array([0, 6, 9])
    q, k, v, do = (r.standard_normal((9, h, 4)) for h in (2, 1, 1, 2))

    def loss(q, k, v):
        return (R.packed(q, k, v, starts, True, 0.5)[0] * do).sum()

    res, _ = R.packed_grad(q, k, v, starts, do, True, 0.5, "bfloat16")
    for i, x in enumerate((q, k, v)):
        for at in [(0, 0, 1), (4, 0, 2), (8, 0, 3)]:
            args = [q, k, v]
            lo, hi = x.copy(), x.copy()
            lo[at] -= 1e-5
            hi[at] += 1e-5
            d = (loss(*args[:i], hi, *args[i + 1:]) - loss(*args[:i], lo, *args[i + 1:])) / 2e-5
            assert abs(d - res[i][at]) < 1e-7


def test_packed_call_is_repeatable(gpu):
    r = np.random.default_rng(4)
    starts = ints([0, 400, 450, 999])
    (q, _), (k, _), (v, _) = make(r, 999, 8, 2, 128, "bfloat16")
    first = None
    for _ in range(3):
        out, stats = O.packedAttention(q, k, v, starts, withLse=True)
        got = [E.toHost(t) for t in (out, *stats, *O.packedAttentionGrad(q, k, v, starts, out, stats, q))]
        for a, b in zip(got, first or got):
            np.testing.assert_array_equal(a, b)
        first = first or got
