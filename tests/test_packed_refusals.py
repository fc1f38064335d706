"""Arguments that the packed and paged operators refuse, checked before any device work (the
operands here have no storage), and the float64 forms that the GPU tests compare with."""
import numpy as np
import pytest

import packed_ref as R
from rew_amd import ops as O
from rew_amd.eager import Device, DType, Tensor, TensorError

BF, F32, I32 = DType.BFLOAT16, DType.FLOAT32, DType.INT32
DEV = Device("mi355x", 0)


def t(dtype, *shape):
    return Tensor(None, dtype, shape, DEV)


def refuse(match, fn, *args, **kw):
    with pytest.raises(TensorError, match=match):
        fn(*args, **kw)


Q, K, S = t(BF, 10, 8, 64), t(BF, 10, 2, 64), t(I32, 4)


@pytest.mark.parametrize("match,args,kw", [
    ("one dtype", (Q, K, t(BF, 10, 2, 32), S), {}),
    ("one dtype", (Q, K, t(F32, 10, 2, 64), S), {}),
    ("one dtype", (Q, t(BF, 10, 128), t(BF, 10, 128), S), {}),
    ("dtype mismatch", (t(F32, 10, 8, 64), K, K, S), {}),
    ("tokens, heads, headDim", (t(BF, 10, 512), K, K, S), {}),
    ("head dims", (t(BF, 10, 8, 128), K, K, S), {}),
    ("do not divide", (t(BF, 10, 7, 64), K, K, S), {}),
    ("do not divide", (t(BF, 10, 8, 64), t(BF, 10, 0, 64), t(BF, 10, 0, 64), S), {}),
    ("tokens", (t(BF, 11, 8, 64), K, K, S), {}),
    ("starts must be int32", (Q, K, K, t(DType.INT64, 4)), {}),
    ("starts must be int32", (Q, K, K, t(I32, 4, 1)), {}),
    ("at least one", (Q, K, K, t(I32, 0)), {}),
    ("scale", (Q, K, K, S), {"scale": -1.0}),
    ("scale", (Q, K, K, S), {"scale": float("nan")}),
    ("scale", (Q, K, K, S), {"scale": float("inf")}),
    ("device", (Q, K, Tensor(None, BF, K.shape, Device("mi355x", 1)), S), {}),
])
def test_packed_refusals(match, args, kw):
    refuse(match, O.packedAttention, *args, **kw)


def test_packed_grad_refusals():
    lse, rest = t(F32, 10, 8), t(DType.INT8, 10, 8, 64)
    st = O.PackedStats(lse, rest)
    refuse("out must", O.packedAttentionGrad, Q, K, K, S, K, st, Q)
    refuse("gradOut must", O.packedAttentionGrad, Q, K, K, S, Q, st, t(F32, 10, 8, 64))
    refuse("lse must", O.packedAttentionGrad, Q, K, K, S, Q, (t(F32, 8, 10), rest), Q)
    refuse("lse must", O.packedAttentionGrad, Q, K, K, S, Q, (t(BF, 10, 8), rest), Q)
    refuse("rest must", O.packedAttentionGrad, Q, K, K, S, Q, (lse, Q), Q)
    refuse("rest must", O.packedAttentionGrad, Q, K, K, S, Q, (lse, t(DType.INT8, 10, 512)), Q)
    refuse("head dims", O.packedAttentionGrad, t(BF, 10, 8, 32), K, K, S, Q, st, Q)


P = t(BF, 30, 2, 16, 64)


def test_paged_refusals():
    tab, st, ln = t(I32, 3, 9), S, t(I32, 3)
    refuse("pages, kvHeads", O.pagedAttention, Q, P, t(BF, 30, 2, 16, 32), tab, st, ln)
    refuse("page size 12", O.pagedAttention, Q, *[t(BF, 30, 2, 12, 64)] * 2, tab, st, ln)
    refuse("page size 0", O.pagedAttention, Q, *[t(BF, 30, 2, 0, 64)] * 2, tab, st, ln)
    refuse("dtype mismatch", O.pagedAttention, t(DType.FLOAT16, 10, 8, 64), P, P, tab, st, ln)
    refuse("blockTable", O.pagedAttention, Q, P, P, t(I32, 27), st, ln)
    refuse("starts", O.pagedAttention, Q, P, P, tab, t(I32, 3), ln)
    refuse("lens", O.pagedAttention, Q, P, P, tab, st, t(I32, 4))
    refuse("maxNew", O.pagedAttention, Q, P, P, tab, st, ln, maxNew=-1)


def test_block_table_refusals():
    c, n, tab, fr = t(I32, 3), t(I32, 3), t(I32, 3, 9), t(I32, 5)
    refuse("page size 24", O.pagedBlockTables, c, n, tab, fr, 24, 5)
    refuse("cachedLens", O.pagedBlockTables, t(I32, 2), n, tab, fr, 16, 5)
    refuse("newLens", O.pagedBlockTables, c, t(F32, 3), tab, fr, 16, 5)
    refuse("freePages", O.pagedBlockTables, c, n, tab, t(I32, 5, 1), 16, 5)
    refuse("tokens", O.pagedBlockTables, c, n, tab, fr, 16, -1)


def test_cache_write_refusals():
    k, s = t(BF, 10, 2, 64), t(I32, 10)
    refuse("one dtype", O.pagedCacheWrite, P, P, k, t(BF, 9, 2, 64), s)
    refuse("do not fit", O.pagedCacheWrite, P, P, *[t(BF, 10, 4, 64)] * 2, s)
    refuse("do not fit", O.pagedCacheWrite, P, P, *[t(F32, 10, 2, 64)] * 2, s)
    refuse("slots", O.pagedCacheWrite, P, P, k, k, t(I32, 11))
    refuse("page size 10", O.pagedCacheWrite, *[t(BF, 30, 2, 10, 64)] * 2, k, k, s)


def test_no_traced_form():
    from rew_amd import jit as J
    with pytest.raises(TensorError, match="eager only"):
        J.lazy(lambda a: [O.packedAttention(a[0], a[1], a[1], a[2])]).call([Q, K, S])


def test_reference_forms_agree():
    """packed_ref's pages, tables and dense attention say the same of one prompt."""
    r = np.random.default_rng(0)
    k, v, q = (r.standard_normal((21, h, 8)) for h in (2, 2, 4))
    table, slots, pos, starts, lens, taken = R.block_tables(
        [0, 0], [13, 8], np.full((2, 5), -1), [9, 4, 7, 1, 3, 0, 8], 4, 21)
    kp, vp = np.full((10, 2, 4, 8), np.nan), np.full((10, 2, 4, 8), np.nan)
    for t_, s in enumerate(slots):
        kp[s // 4, :, s % 4], vp[s // 4, :, s % 4] = k[t_], v[t_]
    want, _, _ = R.packed(q, k, v, starts, True, 0.3)
    for i in range(2):
        kk, there = R.gather_pages(kp, table[i], lens[i])
        vv, _ = R.gather_pages(vp, table[i], lens[i])
        a, b = starts[i], starts[i + 1]
        got = R.attend(q[a:b], kk, vv, 0, True, 0.3, there)[0]
        np.testing.assert_allclose(got, want[a:b], rtol=1e-12, atol=1e-12)
    assert taken[0] == 6 and list(pos) == list(range(13)) + list(range(8))
