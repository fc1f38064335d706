"""Arguments that embeddings, layer norm and the cross entropy refuse, checked before any device
work (the operands here have no storage)."""
import pytest

from rew_amd import ops as O
from rew_amd.eager import Device, DType, Tensor, TensorError

BF, F16, F32, F64, I32 = (DType.BFLOAT16, DType.FLOAT16, DType.FLOAT32, DType.FLOAT64,
                          DType.INT32)
DEV = Device("mi355x", 0)


def t(dtype, *shape, device=DEV):
    return Tensor(None, dtype, shape, device)


def refuse(match, fn, *args, **kw):
    with pytest.raises(TensorError, match=match):
        fn(*args, **kw)


W, IDS = t(BF, 100, 64), t(I32, 7)


@pytest.mark.parametrize("match,args", [
    (r"\[vocab, embed\]", (t(BF, 100), IDS)), ("only float32", (t(F64, 100, 64), IDS)),
    ("int32", (W, t(DType.INT64, 7))), ("int32", (W, t(F32, 7))),
    ("1 to 2\\^20", (t(BF, 100, 0), IDS)), ("1 to 2\\^20", (t(BF, 1, 2 ** 20 + 1), IDS)),
    ("scale", (W, IDS, float("nan"))), ("scale", (W, IDS, 1e39)),
    ("device", (W, t(I32, 7, device=Device("mi355x", 1)))),
])
def test_embedding(match, args):
    refuse(match, O.embedding, *args)


@pytest.mark.parametrize("match,args", [
    ("gradOut", (IDS, t(BF, 8, 64), 100)), ("gradOut", (IDS, t(BF, 7), 100)),
    ("gradOut", (t(I32, 2, 7), t(BF, 14, 64), 100)), ("gradOut", (IDS, t(BF), 100)),
    ("only float32", (IDS, t(I32, 7, 64), 100)), ("int32", (t(BF, 7), t(BF, 7, 64), 100)),
    ("vocab", (IDS, t(BF, 7, 64), 0)), ("vocab", (IDS, t(BF, 7, 64), -5)),
    ("scale", (IDS, t(BF, 7, 64), 100, float("inf"))), ("1 to 2\\^20", (IDS, t(BF, 7, 0), 9)),
])
def test_embedding_grad(match, args):
    refuse(match, O.embeddingGrad, *args)


X, G = t(BF, 5, 6, 32), t(F32, 32)


@pytest.mark.parametrize("match,args,kw", [
    ("only float32", (t(F64, 5, 32), t(F64, 32), t(F64, 32)), {}),
    ("gamma must have", (X, t(F16, 32), t(F16, 32)), {}), ("last dims", (X, t(F32, 6), G), {}),
    ("last dims", (X, t(F32), t(F32)), {}), ("last dims", (X, t(F32, 2, 5, 6, 32), G), {}),
    ("at least one", (t(BF, 5, 0), t(F32, 0), t(F32, 0)), {}), ("beta", (X, G, t(BF, 32)), {}),
    ("beta", (X, G, t(F32, 6, 32)), {}), ("eps", (X, G, G), {"eps": 0.0}),
    ("eps", (X, G, G), {"eps": -1.0}), ("eps", (X, G, G), {"eps": 1e-60}),
    ("eps", (X, G, G), {"eps": float("nan")}),
    ("device", (X, G, t(F32, 32, device=Device("mi355x", 1))), {}),
])
def test_layer_norm(match, args, kw):
    refuse(match, O.layerNorm, *args, **kw)


def test_layer_norm_grad():
    m = t(F32, 5, 6)
    st = O.NormStats(m, m)
    refuse("mean", O.layerNormGrad, X, G, (t(F32, 30), m), X)
    refuse("rstd", O.layerNormGrad, X, G, (m, t(BF, 5, 6)), X)
    refuse("gradOut", O.layerNormGrad, X, G, st, t(F32, 5, 6, 32))
    refuse("gradOut", O.layerNormGrad, X, G, st, t(BF, 30, 32))
    refuse("last dims", O.layerNormGrad, X, t(F32, 31), st, X)


H, HW, TG = t(BF, 9, 64), t(BF, 64, 200), t(I32, 9)


@pytest.mark.parametrize("match,args", [
    ("rank 2", (t(BF, 3, 3, 64), HW, TG)), ("rank 2", (H, t(BF, 64), TG)),
    ("dtype mismatch", (H, t(F16, 64, 200), TG)),
    ("only bfloat16", (t(F32, 9, 64), t(F32, 64, 200), TG)), ("differ", (H, HW, TG, True)),
    ("differ", (H, t(BF, 200, 64), TG)), ("1 to 2", (H, t(BF, 64, 0), TG)),
    ("1 to 2", (H, t(BF, 64, 2 ** 21 + 1), TG)),
    ("targets must be int32", (H, HW, t(I32, 8))),
    ("targets must be int32", (H, HW, t(DType.INT64, 9))),
    ("targets must be int32", (H, HW, t(I32, 9, 1))),
    ("device", (H, HW, t(I32, 9, device=Device("mi355x", 1)))),
])
def test_cross_entropy(match, args):
    refuse(match, O.linearCrossEntropy, *args)


def test_cross_entropy_grad():
    f = t(F32, 9)
    refuse("lse", O.linearCrossEntropyGrad, H, HW, TG, t(F32, 8), f)
    refuse("lse", O.linearCrossEntropyGrad, H, HW, TG, t(BF, 9), f)
    refuse("gradLoss", O.linearCrossEntropyGrad, H, HW, TG, f, t(F32))
    refuse("gradLoss", O.linearCrossEntropyGrad, H, HW, TG, f, t(BF, 9))
    refuse("differ", O.linearCrossEntropyGrad, H, HW, TG, f, f, True)


def test_no_traced_form():
    from rew_amd import jit as J
    with pytest.raises(TensorError, match="eager only"):
        J.lazy(lambda a: [O.embedding(a[0], a[1])]).call([W, IDS])
