"""GPU checks of embeddings, layer norm, packed attention and the loss together, as a training
step uses them: every stage against float64 on the values that the stage before left, replayed
plans, captured graphs, operands that are views, sizes past 32-bit offsets and the library's own
refusals."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import ends_ref as R
import packed_ref as P
from ends_ref import host, ints, tensor
from rew_amd import eager as E
from rew_amd import nn
from rew_amd import ops as O
from rew_amd.eager import DType, EagerError
from test_gpu_capture import _capture

EPS = float(np.float32(1e-5))
V, EMB, HEADS, SCALE = 300, 128, 2, 128 ** 0.5
STARTS = [0, 40, 41, 97]
T = STARTS[-1] + 3  # the last tokens belong to no document


def model(r, dtype, tied):
    def norm():
        return nn.LayerNorm(tensor(1 + 0.2 * r.standard_normal(EMB), "float32")[0],
                            tensor(0.2 * r.standard_normal(EMB), "float32")[0], [EMB])
    emb = nn.Embedding(tensor(r.standard_normal((V, EMB)) / EMB ** 0.5, dtype)[0])
    head = None if tied else nn.LossHead(
        tensor(r.standard_normal((EMB, V)) * 2 / EMB ** 0.5, dtype)[0])
    return emb, norm(), norm(), head


def batch(r):
    ids, targets = r.integers(0, V, T), r.integers(0, V, T)
    ids[STARTS[-1]:], targets[STARTS[-1]:] = -1, -1
    targets[[39, 40, 96]] = -1  # the last token of a document has no next one
    grad = np.where(targets < 0, 0.0, r.uniform(0.5, 1.5, T) / T).astype(np.float32)
    return ids, targets, grad


def step(m, ids, targets, grad):
    """One training step's forward and backward pass: everything it makes, by name."""
    emb, n1, n2, head = m
    out = emb if head is None else head
    s = {"x": emb.rows(ids, SCALE)}
    s["h"], st1 = n1.forwardTrain(s["x"])
    s["q"] = O.reshape(s["h"], [T, HEADS, EMB // HEADS])
    starts = ints(STARTS)
    s["a"], sta = O.packedAttention(s["q"], s["q"], s["q"], starts, withLse=True)
    s["r"] = O.add(s["x"], O.reshape(s["a"], [T, EMB]))
    s["y"], st2 = n2.forwardTrain(s["r"])
    s["loss"], s["lse"] = out.loss(s["y"], targets)
    s["gy"], s["gw"] = out.lossGrad(s["y"], targets, s["lse"], grad)
    s["gr"], s["gg2"], s["gb2"] = n2.grad(s["r"], st2, s["gy"])
    s["ga"] = O.reshape(s["gr"], [T, HEADS, EMB // HEADS])
    s["gq"], s["gk"], s["gv"] = O.packedAttentionGrad(s["q"], s["q"], s["q"], starts, s["a"], sta,
                                                      s["ga"])
    s["gh"] = O.reshape(O.add(O.add(s["gq"], s["gk"]), s["gv"]), [T, EMB])
    s["gx1"], s["gg1"], s["gb1"] = n1.grad(s["x"], st1, s["gh"])
    s["gx"] = O.add(s["gr"], s["gx1"])
    s["gt"] = emb.rowsGrad(ids, s["gx"], SCALE)
    return s


def check_stages(m, s, ids, targets, grad, dtype):
    emb, n1, n2, head = m
    v = {k: host(t) for k, t in s.items()}
    w = host(emb.weight)
    R.check(s["x"], *R.embedding(w, ids, SCALE, dtype))
    for n, x, y in ((n1, "x", "h"), (n2, "r", "y")):
        R.check(s[y], *R.layer_norm(v[x], host(n.gamma), host(n.beta), EPS, dtype)[0])
    want, _, mag = P.packed(v["q"], v["q"], v["q"], STARTS, True, (EMB // HEADS) ** -0.5)
    R.check(s["a"], want, P.out_bound(want, mag, dtype))
    hw = w.T if head is None else host(head.weight)
    for got, (want, bound) in zip((s["loss"], s["lse"]), R.cross_entropy(v["y"], hw, targets)):
        R.check(got, want, bound)
    (gy, e_gy), (gw, e_gw) = R.cross_entropy_grad(v["y"], hw, targets, grad.astype(np.float64),
                                                  dtype)
    R.check(s["gy"], gy, e_gy)
    R.check(s["gw"], gw.T if head is None else gw, e_gw.T if head is None else e_gw)
    for n, x, dy, names in ((n2, "r", "gy", ("gr", "gg2", "gb2")),
                            (n1, "x", "gh", ("gx1", "gg1", "gb1"))):
        for name, (want, bound) in zip(names, R.layer_norm_grad(v[x], host(n.gamma), EPS, v[dy],
                                                                dtype, "float32")):
            R.check(s[name], want, bound)
    R.check(s["gt"], *R.embedding_grad(ids, v["gx"], V, SCALE, dtype))


@pytest.mark.parametrize("tied", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_training_step(gpu, dtype, tied):
    """Several steps over other documents; from the second on every flush replays its plan."""
    r = np.random.default_rng(7)
    m = model(r, dtype, tied)
    E.clearEagerCache()
    for i in range(3):
        ids, targets, grad = batch(r)
        args = ints(ids), ints(targets), E.fromHost(grad)
        E.sync()
        E.resetStats()
        s = step(m, *args)
        E.sync()
        st = E.stats()
        assert i == 0 or st["flush_plan_hits"] == st["flushes"] > 0
        check_stages(m, s, ids, targets, grad, dtype)


def test_captured_training_steps(gpu):
    """Two graphs of the same step over other inputs, replayed in turn with eager steps between
    them: each replay gives the eager result's bits."""
    r = np.random.default_rng(8)
    m = model(r, "bfloat16", False)
    names = ("loss", "gy", "gw", "gg1", "gb2", "gt")
    inputs, wants, graphs = [], [], []
    for _ in range(2):
        ids, targets, grad = batch(r)
        inputs.append((ints(ids), ints(targets), E.fromHost(grad)))
        s = step(m, *inputs[-1])
        wants.append([E.toHost(s[n]) for n in names])
        del s
    for a in inputs:
        graphs.append(_capture(lambda: step(m, *a)))
    for turn in range(3):
        for i in (0, 1):
            graphs[i][0]()
            E.sync()
            for n, w in zip(names, wants[i]):
                np.testing.assert_array_equal(E.toHost(graphs[i][2][n]), w)
            s = step(m, *inputs[1 - i])
            for n, w in zip(names, wants[1 - i]):
                np.testing.assert_array_equal(E.toHost(s[n]), w)
        graphs[0][0]()
        graphs[1][0]()
        E.sync()
        for i in (0, 1):
            for n, w in zip(names, wants[i]):
                np.testing.assert_array_equal(E.toHost(graphs[i][2][n]), w)


FORMS = {  # (tokens, embed, vocab): small and large tiles, a vocabulary in pieces, sums in parts
    "small": (100, 64, 500), "long_k": (3000, 8, 40), "large": (600, 512, 3000),
    "pieces": (2100, 64, 33001),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("tied", [False, True])
def test_captured_losses(gpu, form, tied):
    T_, H, V_ = FORMS[form]
    r = np.random.default_rng(9)
    x = tensor(r.standard_normal((T_, H)), "bfloat16")[0]
    w = tensor(r.standard_normal((V_, H) if tied else (H, V_)), "bfloat16")[0]
    t, g = ints(r.integers(-1, V_, T_)), E.fromHost(r.random(T_).astype(np.float32))

    def call():
        loss, lse = O.linearCrossEntropy(x, w, t, tied, withLse=True)
        return [loss, lse, *O.linearCrossEntropyGrad(x, w, t, lse, g, tied)]

    want = [E.toHost(o) for o in call()]
    replay, _, out = _capture(call)
    for _ in range(3):
        replay()
        between = call()
        E.sync()
        for o, b, k in zip(out, between, want):
            np.testing.assert_array_equal(E.toHost(o), k)
            np.testing.assert_array_equal(E.toHost(b), k)


@pytest.mark.parametrize("tokens,vocab,width", [(300, 700, 40), (3000, 34001, 1003)])
def test_captured_table_gradient(gpu, tokens, vocab, width):
    """Rows of many tokens, of few and of none, in a small table and in one that is cleared as
    a whole."""
    r = np.random.default_rng(11)
    ids = ints(np.floor(np.exp(r.uniform(0, np.log(vocab), tokens))).astype(np.int64) - 1)
    g = tensor(r.standard_normal((tokens, width)), "bfloat16")[0]

    def call():
        return [O.embeddingGrad(ids, g, vocab, 2.0)]

    want = E.toHost(call()[0])
    replay, _, out = _capture(call)
    for _ in range(3):
        replay()
        between = call()
        E.sync()
        np.testing.assert_array_equal(E.toHost(out[0]), want)
        np.testing.assert_array_equal(E.toHost(between[0]), want)


def test_operands_that_are_views(gpu):
    """Slices, transposes and sums that no launch has made yet."""
    r = np.random.default_rng(10)
    big, bigh = tensor(r.standard_normal((40, 96)), "bfloat16")
    wt, wth = tensor(r.standard_normal((50, 64)), "bfloat16")
    x, xh = O.slice_(big, [5, 16], [35, 80]), bigh[5:35, 16:80]
    t = r.integers(-1, 50, 30)
    w = O.transpose(wt, [1, 0])
    loss, lse = O.linearCrossEntropy(x, w, ints(t), withLse=True)
    R.check(loss, *R.cross_entropy(xh, wth.T, t)[0])
    g = E.fromHost(np.ones(30, np.float32))
    half = O.mul(g, O.broadcastTo(O.scalarF32(0.5), [30], []))
    for got, (want, bound) in zip(O.linearCrossEntropyGrad(x, w, ints(t), lse, half),
                                  R.cross_entropy_grad(xh, wth.T, t, np.full(30, 0.5),
                                                       "bfloat16")):
        R.check(got, want, bound)
    ga, gah = tensor(r.standard_normal(64), "float32")
    y, st = O.layerNorm(x, ga, ga, withStats=True)
    R.check(y, *R.layer_norm(xh, gah, gah, EPS, "bfloat16")[0])
    for got, (want, bound) in zip(O.layerNormGrad(x, ga, st, x), R.layer_norm_grad(
            xh, gah, EPS, xh, "bfloat16", "float32")):
        R.check(got, want, bound)
    ids = r.integers(-1, 64, (6, 5))
    it = O.reshape(ints(ids), [30])
    R.check(O.embedding(w, it), *R.embedding(wth.T, ids.reshape(-1), 1.0, "bfloat16"))
    R.check(O.embeddingGrad(it, x, 70), *R.embedding_grad(ids, xh, 70, 1.0, "bfloat16"))


def test_weight_past_32_bit_offsets(gpu):
    """A weight of nearly 2^32 bytes, the product of two vectors of powers of two (exact)."""
    H, V_, T_ = 4096, 500000, 3
    r = np.random.default_rng(11)
    a = 2.0 ** r.integers(-8, -4, H) * r.choice([-1, 1], H)
    b = 2.0 ** r.integers(-2, 2, V_) * r.choice([-1, 1], V_)
    w = O.matmul(tensor(a[:, None], "bfloat16")[0], tensor(b[None], "bfloat16")[0])
    x, xh = tensor(r.standard_normal((T_, H)), "bfloat16")
    t = np.array([V_ - 1, 17, V_ - 77])
    z = (xh @ a)[:, None] * b
    m = z.max(1, keepdims=True)
    lse = (m + np.log(np.exp(z - m).sum(1, keepdims=True)))[:, 0]
    loss, lse_t = O.linearCrossEntropy(x, w, ints(t), withLse=True)
    # (float32 sums of H products below |x| |a| and of V exponentials)
    off = 2 * H * R.U * (np.abs(xh) @ np.abs(a)).max() * 2 + V_ / 8 * R.U
    assert np.abs(host(lse_t) - lse).max() <= off
    assert np.abs(host(loss) - (lse - z[np.arange(T_), t])).max() <= 2 * off
    g = np.array([1.0, 0.5, 2.0])
    dx, dw = O.linearCrossEntropyGrad(x, w, ints(t), lse_t, E.fromHost(g.astype(np.float32)))
    dz = np.exp(z - lse[:, None])
    dz[np.arange(T_), t] -= 1.0
    dz *= g[:, None]
    e_dz = 2.0 ** -7 * np.abs(dz) + 4 * off * np.exp(z - lse[:, None])
    want = np.outer(dz @ b, a)
    bound = np.outer(e_dz @ np.abs(b) + 2 * V_ * R.U * (np.abs(dz) @ np.abs(b)), np.abs(a))
    R.check(dx, want, bound + 2.0 ** -8 * np.abs(want))
    for v0 in (0, V_ - 200):
        got = O.slice_(dw, [H - 40, v0], [H, v0 + 200])
        want = xh[:, H - 40:].T @ dz[:, v0:v0 + 200]
        bound = np.abs(xh[:, H - 40:]).T @ e_dz[:, v0:v0 + 200]
        R.check(got, want, 1.01 * bound + 2.0 ** -7 * np.abs(want))


def test_rows_past_32_bit_offsets(gpu):
    """Layer norm over 4.4e9 bytes of float32, rows of a small table over and over."""
    n, rows = 4096, 270000
    r = np.random.default_rng(12)
    small, sh = tensor(r.standard_normal((7, n)), "float32")
    dsmall, dsh = tensor(r.standard_normal((7, n)), "float32")
    g, gh = tensor(1 + 0.2 * r.standard_normal(n), "float32")
    ids = np.arange(rows) % 7
    x, dy = O.embedding(small, ints(ids)), O.embedding(dsmall, ints(ids))
    y, st = O.layerNorm(x, g, g, withStats=True)
    want, bound = R.layer_norm(sh, gh, gh, EPS, "float32")[0]
    for at in (0, rows - 7):
        k = ids[at:at + 7]
        R.check(O.slice_(y, [at, 0], [at + 7, n]), want[k], bound[k])
    del y
    dx, dg, db = O.layerNormGrad(x, g, st, dy)
    (wx, bx), _, _ = R.layer_norm_grad(sh, gh, EPS, dsh, "float32", "float32")
    k = ids[rows - 7:]
    R.check(O.slice_(dx, [rows - 7, 0], [rows, n]), wx[k], bx[k])
    count = np.bincount(ids)[:, None]
    _, _, _, xh, _, e_xh = R._row(sh, EPS)
    chain = (rows / 256 + 64) * R.U
    R.check(dg, (count * dsh * xh).sum(0),
            (count * np.abs(dsh) * (chain * np.abs(xh) + e_xh)).sum(0) + 1e-6)
    R.check(db, (count * dsh).sum(0), chain * (count * np.abs(dsh)).sum(0) + 1e-6)


@pytest.mark.parametrize("op,shapes,attrs", [
    ("embedding", [("w", 5, 8)], {}), ("embedding", [("w", 5, 8), ("w", 3)], {"scale": "1.0"}),
    ("embedding", [("w", 5, 8), ("i", 3)], {}),
    ("embedding", [("w", 5, 8), ("i", 3)], {"scale": "nan"}),
    ("embedding", [("w", 5), ("i", 3)], {"scale": "1.0"}),
    ("embeddingGrad", [("i", 3), ("w", 4, 8)], {"scale": "1.0", "vocab": "5"}),
    ("embeddingGrad", [("i", 3), ("w", 3, 8)], {"scale": "1.0", "vocab": "0"}),
    ("embeddingGrad", [("i", 3), ("w", 3, 8)], {"scale": "1.0"}),
    ("layerNorm", [("w", 5, 8), ("w", 5), ("w", 5)], {"eps": "1e-5", "stats": "true"}),
    ("layerNorm", [("w", 5, 8), ("w", 8), ("w", 8)], {"eps": "0", "stats": "true"}),
    ("layerNorm", [("w", 5, 8), ("w", 8), ("w", 8)], {"eps": "1e-5", "stats": "yes"}),
    ("layerNorm", [("w", 5, 8), ("h", 8), ("h", 8)], {"eps": "1e-5", "stats": "true"}),
    ("layerNormGrad", [("w", 5, 8), ("w", 8), ("w", 4), ("w", 5), ("w", 5, 8)], {}),
    ("layerNormGrad", [("w", 5, 8), ("w", 8), ("w", 5), ("w", 5), ("w", 40)], {}),
    ("linearCrossEntropy", [("w", 5, 8), ("w", 8, 9), ("i", 5)],
     {"tied": "false", "stats": "true"}),
    ("linearCrossEntropy", [("h", 5, 8), ("h", 8, 9), ("i", 5)],
     {"tied": "true", "stats": "true"}),
    ("linearCrossEntropy", [("h", 5, 8), ("h", 8, 9), ("i", 4)],
     {"tied": "false", "stats": "true"}),
    ("linearCrossEntropy", [("h", 5, 8), ("h", 8, 9), ("i", 5)], {"stats": "true"}),
    ("linearCrossEntropyGrad", [("h", 5, 8), ("h", 8, 9), ("i", 5), ("w", 4), ("w", 5)],
     {"tied": "false"}),
    ("linearCrossEntropyGrad", [("h", 5, 8), ("h", 8, 9), ("i", 5), ("w", 5), ("h", 5)],
     {"tied": "false"}),
])
def test_library_refusals(gpu, op, shapes, attrs):
    """What the library refuses by itself, whatever called it."""
    dt = {"w": DType.FLOAT32, "h": DType.BFLOAT16, "i": DType.INT32}
    ins = [E.empty(dt[s[0]], s[1:]) for s in shapes]
    with pytest.raises(EagerError):
        E.dispatchEager(op, ins, list(attrs.items()))
