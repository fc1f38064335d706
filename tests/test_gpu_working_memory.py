"""GPU checks of what the sequence and training ops hold in device memory: their working memory is
returned behind the launch, whatever becomes of the result; a captured call keeps its own."""
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from ends_ref import ints, tensor
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType
from test_gpu_capture import _capture

MIB = 1 << 20


def f32(a):
    return E.fromHost(np.asarray(a, np.float32))


def calls():
    """name -> (the call, least bytes of its working memory)."""
    r = np.random.default_rng(0)
    T, H, V = 300, 1000, 20001
    x = tensor(r.standard_normal((T, H)), "bfloat16")[0]
    w = tensor(r.standard_normal((H, V)) / 30, "bfloat16")[0]
    t, g = ints(r.integers(-1, V, T)), f32(r.random(T))
    ids = ints(r.integers(0, 500000, 20000))
    rows = tensor(r.standard_normal((20000, 200)), "bfloat16")[0]
    gamma = f32(np.ones(1000))
    wide = tensor(r.standard_normal((3000, 1000)), "bfloat16")[0]
    q = tensor(r.standard_normal((2000, 16, 64)), "bfloat16")[0]
    starts = ints([0, 500, 501, 1990])
    pages = tensor(r.standard_normal((300, 4, 128, 64)), "bfloat16")[0]
    table = ints(np.arange(300).reshape(2, 150))

    new = tensor(r.standard_normal((40, 16, 64)), "bfloat16")[0]
    begins, lens = ints([0, 30, 40]), ints([19000, 9000])

    def loss_grad():
        loss, lse = O.linearCrossEntropy(x, w, t, withLse=True)
        return [*O.linearCrossEntropyGrad(x, w, t, lse, g), loss, lse]

    def norm_grad():
        y, st = O.layerNorm(wide, gamma, gamma, withStats=True)
        return [*O.layerNormGrad(wide, gamma, st, wide), y, *st]

    def attention_grad():
        out, st = O.packedAttention(q, q, q, starts, withLse=True)
        return [*O.packedAttentionGrad(q, q, q, starts, out, st, q), out, *st]

    return {
        "loss": (lambda: [O.linearCrossEntropy(x, w, t)], 2 * H * 16384),
        "loss_grad": (loss_grad, 2 * H * V),
        "embedding_grad": (lambda: [O.embeddingGrad(ids, rows, 500000)], 4 * 500000),
        "norm_grad": (norm_grad, 8 * 1000 * 128),
        "packed_grad": (attention_grad, 8 * 2000 * 16),
        "paged": (lambda: [O.pagedAttention(new, pages, pages, table, begins, lens)], MIB),
    }


def held(res):
    """The bytes of result tensors as the allocator rounds them."""
    total = 0
    for t in res:
        n = int(np.prod(t.shape)) * {DType.FLOAT32: 4, DType.INT8: 1}.get(t.dtype, 2)
        total += (n + 511) // 512 * 512 if n <= MIB else (n + 2 * MIB - 1) // (2 * MIB) * 2 * MIB
    return total


NAMES = ["loss", "loss_grad", "embedding_grad", "norm_grad", "packed_grad", "paged"]


@pytest.fixture(scope="module")
def made(gpu):
    return calls()


def in_use():
    E.sync()
    return E.stats()["bytes_in_use"]


@pytest.mark.parametrize("name", NAMES)
def test_results_hold_no_working_memory(made, name):
    """Kept results of several calls, the first recorded and the others replayed from its plan.
    (A reused block may be a quarter larger than asked for; a small constant is cached.)"""
    call, _ = made[name]
    E.clearEagerCache()
    call()
    before, kept = in_use(), []
    for i in range(1, 5):
        if i == 1:
            E.clearEagerCache()
        kept.append(list(call()))
        size = held([t for res in kept for t in res])
        assert in_use() - before <= 1.25 * size + 8192, i


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("recorded", [False, True])
def test_captured_calls_keep_theirs(made, name, recorded):
    """A graph that records the plan, and one that replays an eager call's: replays between eager
    calls, whose working memory is the same size, give the eager results' bits."""
    call, least = made[name]
    E.clearEagerCache()
    want = [E.toHost(t) for t in call()]
    if recorded:
        E.clearEagerCache()
    keep = call() if not recorded else None
    before = in_use()
    replay, _, out = _capture(call)
    assert in_use() - before >= held(out) + least
    del keep
    for _ in range(3):
        replay()
        between = call()
        E.sync()
        for o, b, k in zip(out, between, want):
            np.testing.assert_array_equal(E.toHost(o), k)
            np.testing.assert_array_equal(E.toHost(b), k)
        del between, o, b
    del out
    assert in_use() - before <= 8192


@pytest.mark.parametrize("name", NAMES)
def test_op_by_op(made, name):
    call, _ = made[name]
    want = [E.toHost(t) for t in call()]
    before = in_use()
    E.setMode(E.MODE_OP_BY_OP)
    try:
        for _ in range(2):
            got = call()
            for g, w in zip(got, want):
                np.testing.assert_array_equal(E.toHost(g), w)
    finally:
        E.setMode(E.MODE_DEFERRED)
    del g
    assert in_use() - before <= 1.25 * held(got) + 8192


CHILD = r"""
import sys
import numpy as np
sys.path.insert(0, sys.argv[1])
from rew_amd import eager as E, ops as O
from rew_amd.eager import DType
E.installEagerBackend(E.mi355x(0))
r = np.random.default_rng(0)
x = E.fromHost(r.standard_normal((64, 2000)).astype(np.float32), DType.BFLOAT16)
w = E.fromHost(r.standard_normal((2000, 20001)).astype(np.float32), DType.BFLOAT16)  # 80 MB
t = E.fromHost(np.zeros(64, np.int32), DType.INT32)
E.sync()
base = E.stats()["bytes_in_use"]
for _ in range(3):                                # its working memory: 65 MB
    loss = O.linearCrossEntropy(x, w, t)
    try:
        E.toHost(loss)
        sys.exit("no error")
    except E.EagerError as e:
        assert "REW_MI355X_MAX_DEVICE_BYTES" in str(e), e
    del loss
    E.sync()
    assert E.stats()["bytes_in_use"] == base, (E.stats()["bytes_in_use"], base)
v = O.slice_(w, [0, 0], [2000, 1000])
E.sync()
a = E.toHost(O.linearCrossEntropy(x, v, t))
b = E.toHost(O.linearCrossEntropy(x, v, t))
assert np.isfinite(a).all() and (a == b).all()
print("ok")
"""


def test_no_room_for_it(gpu):
    """An error where the limit leaves no room, which leaves nothing behind."""
    env = dict(os.environ, REW_MI355X_MAX_DEVICE_BYTES=str(128 * MIB))
    p = subprocess.run([sys.executable, "-c", CHILD, str(Path(__file__).resolve().parents[1])],
                       env=env, capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and p.stdout.strip().endswith("ok"), p.stderr[-3000:]
