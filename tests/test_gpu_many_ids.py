"""GPU checks of the table's gradient with more workgroups than 2^16, which launches hold in rows:
all sums are of small whole numbers, exact in float32 in any order."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from ends_ref import host, ints
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType, EagerError


@pytest.mark.parametrize("tokens,vocab,few", [
    (2 ** 22 + 700, 1000, 1000),      # windows of the order, rows of many tokens
    (2 ** 20, 2 ** 25 + 1025, 2 ** 25 + 1025),  # rows of the sort, and places of a cleared table
    (2 ** 22 + 65, 2 ** 25 - 3, 40),  # both, and rows that go on over many windows
])
def test_many_workgroups(gpu, tokens, vocab, few):
    r = np.random.default_rng(tokens)
    ids = r.integers(-1, few, tokens)
    ids[:3] = vocab - 1
    g = r.integers(-2, 3, tokens).astype(np.float32)
    want = np.bincount(np.where(ids < 0, vocab, ids), g, vocab + 1)[:vocab]
    got = O.embeddingGrad(ints(ids), E.fromHost(g[:, None]), vocab, 2.0)
    np.testing.assert_array_equal(host(got)[:, 0], 2.0 * want)


def test_library_refusal(gpu):
    ids, g = E.empty(DType.INT32, (2 ** 30,)), E.empty(DType.BFLOAT16, (2 ** 30, 1))
    with pytest.raises(EagerError, match="2\\^30 ids"):
        E.dispatchEager("embeddingGrad", [ids, g], [("vocab", "5"), ("scale", "1.0")])
