"""Scales that float32 does not hold: refused, also one that would underflow to 0, which stands
for 1 / sqrt(headDim)."""
import numpy as np
import pytest

import packed_ref as R
from rew_amd import ops as O
from rew_amd.eager import Device, DType, EagerError, Tensor, TensorError

BAD = [1e-50, 5e-324, 1e39, 1e300, -1e-50, float("nan"), float("inf")]


def t(dtype, *shape):
    return Tensor(None, dtype, shape, Device("mi355x", 0))


@pytest.mark.parametrize("scale", BAD)
def test_refused(scale):
    q, i = t(DType.BFLOAT16, 4, 2, 64), lambda n: t(DType.INT32, n)
    pages = [t(DType.BFLOAT16, 3, 2, 16, 64)] * 2
    st = O.PackedStats(t(DType.FLOAT32, 4, 2), t(DType.INT8, 4, 2, 64))
    for call in (lambda: O.packedAttention(q, q, q, i(2), scale=scale),
                 lambda: O.packedAttentionGrad(q, q, q, i(2), q, st, q, scale=scale),
                 lambda: O.pagedAttention(q, *pages, t(DType.INT32, 1, 3), i(2), i(1),
                                          scale=scale)):
        with pytest.raises(TensorError, match="scale"):
            call()


def test_sent_as_it_is():
    for scale, text in ((0.0, "0.0"), (0, "0.0"), (0.125, "0.125"), (1, "1.0"),
                        (np.float32(0.1), "0.10000000149011612")):
        assert dict(O._attn_attrs("op", True, scale))["scale"] == text


@pytest.mark.gpu
@pytest.mark.parametrize("scale", ["1e-50", "0x1p-200", "1e39", "nan", "-1", "", "1x"])
def test_refused_by_the_library(gpu, scale):
    x = gpu.empty(DType.BFLOAT16, (4, 2, 64))
    starts = gpu.fromHost(np.array([0, 4], np.int32))
    with pytest.raises((EagerError, TensorError), match="scale"):
        gpu.executeMi355xOp("packedAttention", [x, x, x, starts],
                            [("causal", "true"), ("scale", scale), ("stats", "false")])


@pytest.mark.gpu
def test_least_scale(gpu):
    """The least positive float32 is a scale: all scores 0, rows the means of what they see."""
    from test_gpu_packed import check, ints, make
    (q, _), (k, _), (v, vh) = make(np.random.default_rng(0), 70, 2, 2, 64, "bfloat16")
    out = O.packedAttention(q, k, v, ints([0, 70]), scale=2.0 ** -149)
    mean, mag = (np.cumsum(x, 0) / np.arange(1, 71)[:, None, None] for x in (vh, np.abs(vh)))
    check(out, mean, R.out_bound(mean, mag, "bfloat16"))
