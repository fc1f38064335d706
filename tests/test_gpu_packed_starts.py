"""GPU checks of starts that fall: a value below an earlier one counts as that one, so no row
belongs to two sequences and no launch has more tiles than the host has counted."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from rew_amd import eager as E
from rew_amd import ops as O
from test_gpu_packed import DTYPES, ints, make, tensor
from test_gpu_paged import paged_call, paged_case


def falling(kind, T, n):
    """n + 1 starts over T rows and what they count as."""
    s = np.zeros(n + 1, np.int64)
    if kind == "alternate":
        s[1::2] = T
    elif kind == "back":
        s = np.random.default_rng(n).integers(-T // 2, T + T // 2, n + 1)
    else:  # one drop in the middle
        s = np.linspace(0, T, n + 1).astype(np.int64)
        s[n // 2] = 0
    return s, np.maximum.accumulate(np.clip(s, 0, T))


KINDS = ["alternate", "back", "drop"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [3, 61, 150])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_packed(gpu, kind, n, dtype, causal):
    T = 400
    r = np.random.default_rng(n)
    (q, _), (k, _), (v, _) = make(r, T, 4, 2, 64, dtype)
    do, _ = tensor(r.standard_normal((T, 4, 64)), dtype)

    def run(starts):
        s = ints(starts)
        out, stats = O.packedAttention(q, k, v, s, causal=causal, withLse=True)
        return [out, *stats, *O.packedAttentionGrad(q, k, v, s, out, stats, do, causal=causal)]

    for g, w in zip(*map(run, falling(kind, T, n))):
        np.testing.assert_array_equal(E.toHost(g), E.toHost(w))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [3, 61, 150])
@pytest.mark.parametrize("T,width,hint", [(20, None, 1), (20, 400, 1), (300, None, 0),
                                          (300, 400, 0)],
                         ids=["few", "few_wide", "chunks", "chunks_wide"])
def test_paged(gpu, kind, n, T, width, hint):
    r = np.random.default_rng(n + T)
    c = paged_case(r, [T] + [0] * (n - 1), [int(x) for x in r.integers(T, 1600, n)], 8, 2, 64, 16,
                   "bfloat16", width=width)
    got = []
    for starts in falling(kind, T, n):
        c["starts"] = starts
        got.append(E.toHost(paged_call(c, maxNew=hint)))
    np.testing.assert_array_equal(*got)
