"""GPU checks of the gradients beside large finite values: what another sequence, another KV
head or an unseen row holds takes no bits of a result, although float16 stores dS scaled."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from test_gpu_packed import DTYPES, ints, make, tensor

# a float16 result below 2^-14 is rounded to a multiple of 2^-24
TINY = 2.0 ** -25


def grads(x, starts, dtype, causal=True):
    q, k, v, do = (tensor(y, dtype)[0] for y in x)
    out, stats = O.packedAttention(q, k, v, ints(starts), causal=causal, withLse=True)
    got = O.packedAttentionGrad(q, k, v, ints(starts), out, stats, do, causal=causal)
    return [E.toHostF32(g).astype(np.float64) for g in got]


def case(seed, T, H, Hkv, D, dtype, size):
    r = np.random.default_rng(seed)
    x = [h for _, h in make(r, T, H, Hkv, D, dtype)]
    return x + [tensor(r.standard_normal((T, H, D)) * size, dtype)[1]]


def close(got, want, bnd, at):
    assert np.isfinite(got[at]).all()
    over = np.abs(got[at] - want[at]) - bnd[at] - TINY
    assert over.max() <= 0, over.max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 32), (6, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("which", [2, 3], ids=["v", "do"])
@pytest.mark.parametrize("value", [1e2, 1e3, 6e4])
def test_other_sequences(gpu, dtype, H, Hkv, D, causal, which, value):
    starts = [0, 70, 370, 441]
    x = case(D, 441, H, Hkv, D, dtype, 1e-3)
    want, bnd = R.packed_grad(*x[:3], starts, x[3], causal, D ** -0.5, dtype)
    x[which][[5, 69, 400], 0, 7] = tensor([value], dtype)[1]
    for g, w, b in zip(grads(x, starts, dtype, causal), want, bnd):
        close(g, w, b, slice(70, 370))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("which", [2, 3], ids=["v", "do"])
def test_other_heads(gpu, dtype, causal, which):
    H, Hkv, D, starts = 6, 3, 64, [0, 200, 300]
    x = case(1, 300, H, Hkv, D, dtype, 1e-3)
    want, bnd = R.packed_grad(*x[:3], starts, x[3], causal, 0.125, dtype)
    x[which][::17, 2 if which == 2 else 4, 7] = tensor([6e4], dtype)[1]
    for g, w, b in zip(grads(x, starts, dtype, causal), want, bnd):
        close(g, w, b, np.s_[:, :g.shape[1] // 3 * 2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,Hkv,D", [(4, 4, 32), (8, 2, 64), (4, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("at", [0, 1, 40, 130, 255, 299])
def test_unseen_rows(gpu, dtype, H, Hkv, D, at):
    """A large V reaches the rows from its own on, a large gradOut the keys up to its own."""
    starts = [0, 300, 333]
    for which in (2, 3):
        x = case(at, 333, H, Hkv, D, dtype, 1e-3)
        want, bnd = R.packed_grad(*x[:3], starts, x[3], True, D ** -0.5, dtype)
        x[which][at, :, 3] = tensor([6e4], dtype)[1]
        got = grads(x, starts, dtype)
        rest = np.r_[0:at, 300:333] if which == 2 else np.r_[0:at, at + 1:333]
        close(got[0], want[0], bnd[0], rest)
        for i in (1, 2):
            close(got[i], want[i], bnd[i], np.r_[at + 1:333] if which == 3 else np.r_[300:333])


@pytest.mark.parametrize("causal", [True, False])
def test_row_of_its_own_size(gpu, causal):
    """Rows of one sequence whose gradients differ by orders of magnitude: each row's dQ."""
    starts, D = [0, 260], 64
    x = case(3, 260, 4, 2, D, "float16", 1.0)
    size = 10.0 ** np.random.default_rng(0).integers(-4, 4, 260)
    x[3] = tensor(x[3] * size[:, None, None], "float16")[1]
    want, bnd = R.packed_grad(*x[:3], starts, x[3], causal, 0.125, "float16")
    close(grads(x, starts, "float16", causal)[0], want[0], bnd[0], slice(None))


@pytest.mark.parametrize("H,Hkv,D", [(7, 7, 32), (40, 1, 64), (71, 1, 128), (15, 5, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_odd_groups(gpu, H, Hkv, D, causal):
    """Groups that do not divide a block of rows, a large gradient in the document before."""
    starts = [0, 30, 200]
    x = case(H, 200, H, Hkv, D, "float16", 1e-3)
    want, bnd = R.packed_grad(*x[:3], starts, x[3], causal, D ** -0.5, "float16")
    x[3][[0, 29], :, 5] = tensor([6e4], "float16")[1]
    for g, w, b in zip(grads(x, starts, "float16", causal), want, bnd):
        close(g, w, b, slice(30, 200))


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [2, 31, 150, 400])
def test_largest_values(gpu, D, causal, n):
    """gradOut and V of one size and sign in all columns, near float16's largest: dS reaches the
    bound that its factor comes from, D max|gradOut| max|V| + |delta|."""
    r = np.random.default_rng(n + D)
    q, k = (tensor(r.standard_normal((n, h, D)), "float16")[1] for h in (4, 2))
    sign = lambda h: np.broadcast_to(r.choice([-1.0, 1.0], (n, h, 1)), (n, h, D))
    v, do = sign(2) * 6e4, sign(4) * 6e4
    x = [q, k, tensor(v, "float16")[1], tensor(do, "float16")[1]]
    # (dQ = scale dS K below 2^-26 D 3.6e9 2 max|k| < 7e4 / 2: no result overflows)
    scale = 2.0 ** -26 / (D / 32)
    want, bnd = R.packed_grad(*x[:3], [0, n], x[3], causal, scale, "float16")
    t = [tensor(y, "float16")[0] for y in x]
    out, stats = O.packedAttention(*t[:3], ints([0, n]), causal=causal, scale=scale, withLse=True)
    got = O.packedAttentionGrad(*t[:3], ints([0, n]), out, stats, t[3], causal=causal, scale=scale)
    for i in (0, 1):
        g = E.toHostF32(got[i]).astype(np.float64)
        fits = np.abs(want[i]) < 6e4
        assert np.isfinite(g[fits]).all() and fits.mean() > 0.9
        assert (np.abs(g - want[i])[fits] <= bnd[i][fits] + TINY).all()
