"""GPU checks of many sequences: more than a launch takes are refused when they are recorded, and
thousands of empty ones change nothing."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType, EagerError
from test_gpu_packed import check, ints, make
from test_gpu_paged import paged_call, paged_case, paged_want

BF = DType.BFLOAT16


def test_refused_at_once(gpu):
    """By the call itself: what was recorded before is not lost to a launch that fails."""
    before = O.add(ints([1, 2]), ints([3, 4]))
    for n, heads, grad_heads in ((2 ** 20, 1, 1), (2 ** 20 - 2, 16, 8), (2 ** 18, 64, 32)):
        starts = E.empty(DType.INT32, (n + 1,))
        x = E.empty(BF, (4, heads, 32))
        with pytest.raises(EagerError, match="sequences"):
            O.packedAttention(x, x, x, starts)
        g = E.empty(BF, (4, grad_heads, 32))
        st = O.PackedStats(E.empty(DType.FLOAT32, (4, grad_heads)),
                           E.empty(DType.INT8, (4, grad_heads, 32)))
        with pytest.raises(EagerError, match="sequences"):
            O.packedAttentionGrad(g, g, g, starts, g, st, g)
        pages = [E.empty(BF, (2, heads, 16, 32)) for _ in range(2)]
        for hint in (0, 1):
            with pytest.raises(EagerError, match="sequences"):
                O.pagedAttention(x, *pages, E.empty(DType.INT32, (n, 1)), starts,
                                 E.empty(DType.INT32, (n,)), maxNew=hint)
    np.testing.assert_array_equal(E.toHost(before), [4, 6])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_thousands_of_empty_sequences(gpu, dtype):
    T, n = 300, 20000
    r = np.random.default_rng(0)
    (q, _), (k, _), (v, _) = make(r, T, 4, 2, 64, dtype)
    few = np.array([3, 50, 51, 200, 290])
    many = np.sort(np.concatenate([few, r.choice(few, n)]))

    def run(starts):
        s = ints(starts)
        out, stats = O.packedAttention(q, k, v, s, withLse=True)
        return [out, *stats, *O.packedAttentionGrad(q, k, v, s, out, stats, q)]

    for g, w in zip(run(many), run(few)):
        np.testing.assert_array_equal(E.toHost(g), E.toHost(w))


@pytest.mark.parametrize("news,lens,width,hint", [
    ([1, 2, 1], [300, 20, 77], None, 2), ([1, 2, 1], [300, 20, 77], 300, 2),
    ([60, 2, 1], [1900, 20, 77], None, 0)], ids=["short", "wide", "chunks"])
def test_thousands_of_idle_requests(gpu, news, lens, width, hint):
    """Requests without new tokens between those that have some."""
    r = np.random.default_rng(1)
    c = paged_case(r, news, lens, 8, 2, 64, 16, "bfloat16", width=width)
    n, at = 3000, [7, 1500, 2999]
    table = r.integers(-1, 5, (n, c["table"].shape[1]))
    table[at] = c["table"]
    all_lens, all_news = r.integers(0, 900, n), np.zeros(n, int)
    all_lens[at], all_news[at] = lens, news
    d = dict(c, table=table, lens=list(all_lens), starts=np.concatenate([[0], np.cumsum(all_news)]))
    # (so many workgroups, whatever the table's width, that the key tiles of all requests are cut
    # into runs: other orders of the sums than with three requests, within the usual bound)
    want, mag = paged_want(d, True, 0.125)
    check(paged_call(d, maxNew=hint), want, R.out_bound(want, mag, "bfloat16"))
