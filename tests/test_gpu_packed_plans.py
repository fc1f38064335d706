"""GPU checks that steps of the packed and paged operators run from recorded plans: every flush
after a form's first replays, with the results of a fresh lowering.  Outputs here fill their
blocks of memory (multiples of 512 bytes), where an address behind them is another block's."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from rew_amd import eager as E
from rew_amd import nn
from rew_amd import ops as O
from test_gpu_packed import DTYPES, ints, make, tensor
from test_gpu_paged import paged_call, paged_case
from test_gpu_serving import layer_of


def packed(r, dtype):
    (q, _), (k, _), (v, _) = make(r, 128, 4, 2, 64, dtype)
    return lambda: [O.packedAttention(q, k, v, ints([0, 60, 128]))]


def training(r, dtype, T=128):
    (q, _), (k, _), (v, _) = make(r, T, 4, 2, 64, dtype)

    def call():
        out, stats = O.packedAttention(q, k, v, ints([0, T]), withLse=True)
        return [out, *O.packedAttentionGrad(q, k, v, ints([0, T]), out, stats, q)]

    return call


def paged(news, lens, width=None):
    def form(r, dtype):
        c = paged_case(r, news, lens, 32, 8, 128, 16, dtype, width=width)
        return lambda: [paged_call(c)]
    return form


def tables(r, dtype):
    table = r.integers(0, 99, (128, 8))
    return lambda: list(O.pagedBlockTables(ints([3] * 128), ints([1] * 128), ints(table),
                                           ints(np.arange(128)), 4, 128))


FORMS = {
    "packed": packed, "training": training, "nothing": lambda r, d: training(r, d, 0),
    "decode_short": paged([1] * 4, [300, 5, 77, 64]),
    "decode_wide": paged([1] * 4, [300, 5, 77, 64], 300),
    "one_worker": paged([1], [20], 129), "chunks": paged([40, 1, 23], [2000, 300, 23]),
    "tables": tables,
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", FORMS)
def test_replays(gpu, form, dtype):
    r = np.random.default_rng(0)
    E.clearEagerCache()
    for i in range(4):
        call = FORMS[form](r, dtype)
        E.sync()
        E.resetStats()
        got = [E.toHost(t) for t in call()]
        s = E.stats()
        assert s["flushes"] and (i == 0 or s["flush_plan_hits"] == s["flushes"]), (i, s)
        E.clearEagerCache()
        for g, t in zip(got, call()):  # (recorded anew, for the next one to replay)
            np.testing.assert_array_equal(g, E.toHost(t))


def test_decode_step_of_a_layer(gpu, oracle):
    """One token of each request through a decoder layer: every flush replays, the projections
    and the feed-forward beside the attention."""
    R = 5
    layer = layer_of(oracle, 0x5EED0031, 512, 8, 2, 512, 64)[1]
    cache = nn.PagedKVCache.init(64, 2, 16, 64)
    r = np.random.default_rng(1)
    table = ints(r.permutation(64)[:4 * R].reshape(R, 4))
    for i in range(6):
        x = tensor(r.standard_normal((R, 512)), "bfloat16")[0]
        E.sync()
        E.resetStats()
        step = O.pagedBlockTables(ints([i + 2] * R), ints([1] * R), table, ints([0]), 16, R)
        E.toHostF32(layer.forwardPaged(x, cache, step, maxNew=1))
        s = E.stats()
        assert i == 0 or s["flush_plan_hits"] == s["flushes"], (i, s)


@pytest.mark.parametrize("R", [1, 2, 4])
def test_other_lengths_of_few_requests(gpu, R):
    """Lengths of up to 16 bytes are known on the host too, but read on the device: steps that
    differ in them alone replay one plan."""
    r = np.random.default_rng(R)
    c = paged_case(r, [1] * R, [400] * R, 8, 2, 64, 16, "bfloat16", width=30)
    (q, _), (k, _), (v, _) = make(r, 90, 4, 2, 64, "bfloat16")
    results = []
    for i in range(1, 6):
        E.sync()
        E.resetStats()
        c["lens"] = list(r.integers(20, 400, R))
        st = O.pagedBlockTables(ints([n + 500 + i for n in c["lens"]]), ints([i] * R),
                                ints(c["table"]), ints([7 + i]), 16, 8)
        cuts = np.sort(r.integers(0, 91, R + 1))
        out, stats = O.packedAttention(q, k, v, ints(cuts), withLse=True)
        tensors = [paged_call(c), out, *O.packedAttentionGrad(q, k, v, ints(cuts), out, stats, q),
                   st.blockTable, st.slots, st.lens]
        E.flush()
        s = E.stats()
        # (the first two may share the memory of equal lengths in another way)
        assert i < 3 or s["flush_plan_hits"] == s["flushes"], (i, s)
        results.append(([E.toHost(t) for t in tensors], c["lens"], cuts, i))
    for got, lens, cuts, i in results:  # each lowered by itself
        E.clearEagerCache()
        c["lens"] = lens
        out, stats = O.packedAttention(q, k, v, ints(cuts), withLse=True)
        st = O.pagedBlockTables(ints([n + 500 + i for n in lens]), ints([i] * R),
                                ints(c["table"]), ints([7 + i]), 16, 8)
        for g, t in zip(got, [paged_call(c), out,
                              *O.packedAttentionGrad(q, k, v, ints(cuts), out, stats, q),
                              st.blockTable, st.slots, st.lens]):
            np.testing.assert_array_equal(g, E.toHost(t))


def test_scalars_are_told_apart(gpu):
    """A scalar that a launch holds as a constant makes its own plan, also where a sequence op
    reads the same tensor."""
    (q, qh), (k, _), (v, _) = make(np.random.default_rng(0), 4, 2, 2, 32, "bfloat16")
    for i in range(4):
        n = ints([i])
        out = O.packedAttention(q, k, v, n)  # (one start: no sequence)
        x = O.add(O.broadcastTo(n, [6], [0]), O.iota(ints([0]).dtype, [6], 0))
        E.flush()
        np.testing.assert_array_equal(E.toHost(x), i + np.arange(6))
        assert not E.toHostF32(out).any()
