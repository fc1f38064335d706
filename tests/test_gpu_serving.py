"""GPU checks of packed and paged attention as decoder layers use them: prompts and single
tokens through block tables, cache writes, attention and the layer around them.

bf16 layers, as in the other layer tests: <= 2e-2 relative, normwise and max-abs."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import nn
from rew_amd import ops as O
from rew_amd.eager import DType
from test_gpu_capture import _capture
from test_gpu_composites import _llama_params, bf16_close, dev, host
from test_gpu_packed import check, ints, make, tensor
from test_gpu_paged import paged_call, paged_case, paged_want


def layer_of(oracle, seed, E_, nh, nkv, I, positions):
    p, m = _llama_params(oracle, oracle.init_key(seed), E_, nh, nkv, I)
    hd = E_ // nh
    attn = nn.GroupedQueryAttention(m["q"], m["k"], m["v"], m["o"], nh, nkv, hd,
                                    nn.RotaryPositionEncoding.init(hd, positions, 500000.0))
    return p, nn.LlamaDecoderLayer(attn, nn.GatedFeedForward(m["g"], m["u"], m["d"]),
                                   nn.RMSNorm(dev(p["g1"])), nn.RMSNorm(dev(p["g2"])))


def test_layer_over_packed_rows(gpu, oracle):
    """Each sequence of a packed batch gives what the layer gives for it alone."""
    E_, nh, nkv, I, lens = 256, 4, 2, 512, [50, 1, 77, 0, 130]
    p, layer = layer_of(oracle, 0x5EED0011, E_, nh, nkv, I, 256)
    starts = np.concatenate([[0], np.cumsum(lens)])
    x = oracle.round_bf16(oracle.normal_f32(oracle.init_key(3), starts[-1] * E_)
                          .reshape(-1, E_))
    pos = np.concatenate([np.arange(n) for n in lens])
    got = host(layer.forwardPacked(dev(x, DType.BFLOAT16), ints(starts), ints(pos),
                                   causal=False))
    c, s = nn.rope_tables(E_ // nh, 256, 500000.0)
    for a, b in zip(starts[:-1], starts[1:]):
        if b > a:
            want = oracle.llama_layer(x[None, a:b], p, nh, nkv, c, s, 1e-5, False, True, "rms")
            bf16_close(got[a:b], want[0])
            alone = layer.forward(dev(x[None, a:b], DType.BFLOAT16), causal=False)
            bf16_close(got[a:b], host(alone)[0])


@pytest.mark.parametrize("page", [4, 16, 64])
@pytest.mark.parametrize("nh,nkv", [(8, 2), (4, 4), (2, 1)])
def test_serving_run(gpu, oracle, page, nh, nkv):
    """Requests that join and leave: prompts whole and in chunks beside single tokens of
    others; two layers with one block table.  Every row equals the packed layers' over the
    whole sequences."""
    E_, I = 64 * nh, 256
    layers = [layer_of(oracle, 0x5EED0020 + i, E_, nh, nkv, I, 512)[1] for i in range(2)]
    total = {0: 70, 1: 133, 2: 9, 3: 260}
    r = np.random.default_rng(page + nh)
    x = {i: r.standard_normal((n, E_)).astype(np.float32) for i, n in total.items()}
    # (request, new tokens) of each step
    steps = [[(0, 60)], [(0, 1), (1, 100)], [(0, 1), (1, 30), (2, 6)], [(1, 1), (2, 1), (0, 1)]]
    steps += [[(2, 1), (3, 250), (0, 1)], [(3, 1), (1, 1)], [(2, 1), (3, 9)], [(0, 6), (1, 1)]]
    pages = sum(-(-n // page) for n in total.values()) + 2
    caches = [nn.PagedKVCache.init(pages, nkv, page, 64) for _ in layers]
    free, tables, done = list(r.permutation(pages)), {}, dict.fromkeys(total, 0)
    width, out = -(-300 // page), {i: np.zeros((n, E_), np.float32) for i, n in total.items()}
    for step in steps:
        news = [n for _, n in step]
        tab = np.stack([tables.get(i, np.full(width, -1)) for i, _ in step])
        st = O.pagedBlockTables(ints([done[i] for i, _ in step]), ints(news), ints(tab),
                                ints(free), page, sum(news))
        rows = np.concatenate([x[i][done[i]:done[i] + n] for i, n in step])
        h = dev(rows, DType.BFLOAT16)
        for layer, cache in zip(layers, caches):
            h = layer.forwardPaged(h, cache, st, maxNew=max(news))
        got, at = host(h), 0
        free = free[int(E.toHost(st.taken)[0]):]
        for (i, n), row in zip(step, E.toHost(st.blockTable)):
            out[i][done[i]:done[i] + n] = got[at:at + n]
            tables[i], done[i], at = row, done[i] + n, at + n
    lens = [done[i] for i in total]
    assert lens == [70, 133, 9, 260]
    h = dev(np.concatenate(list(x.values())), DType.BFLOAT16)
    starts = ints(np.concatenate([[0], np.cumsum(lens)]))
    pos = ints(np.concatenate([np.arange(n) for n in lens]))
    for layer in layers:
        h = layer.forwardPacked(h, starts, pos)
    bf16_close(np.concatenate(list(out.values())), host(h))


def test_rope_at_positions(gpu):
    """forwardAt equals forward where the positions are those of a dense sequence."""
    rope = nn.RotaryPositionEncoding.init(64, 96, 10000.0)
    x = np.random.default_rng(0).standard_normal((50, 3, 64)).astype(np.float32)
    want = host(rope.forward(dev(x.transpose(1, 0, 2)), 7)).transpose(1, 0, 2)
    got, twice = map(host, rope.forwardAt([dev(x), dev(2 * x[:, :1])], ints(np.arange(7, 57))))
    np.testing.assert_array_equal(twice, 2 * got[:, :1])
    np.testing.assert_allclose(got, want, rtol=0, atol=4 * 2.0 ** -23 * np.abs(x).max())
    last, far = (host(rope.forwardAt([dev(x)], ints(np.full(50, p)))[0]) for p in (95, 1000))
    np.testing.assert_array_equal(far, last)


def _replays(capture, other, times=4):
    """The captured call's results after each replay, eager work and a wait between them."""
    replay, _, outs = capture
    got = []
    for _ in range(times):
        other()
        E.sync()
        replay()
        E.sync()
        got.append([E.toHostF32(o) for o in outs])
    return got


@pytest.mark.parametrize("news,lens,width", [([1, 1, 1], [300, 5, 77], None),
                                             ([1, 3, 1], [3000, 5, 700], 300),
                                             ([300, 1, 40], [2500, 90, 300], None)],
                         ids=["short", "runs", "chunks"])
def test_captured_step(gpu, news, lens, width):
    """A serving step (tables, write, attention) captured and replayed between eager steps of
    other sizes, and two captured steps in turn."""
    r = np.random.default_rng(len(news))
    cases = [paged_case(r, news, lens, 8, 2, 64, 16, "bfloat16", width=width),
             paged_case(r, [2, 60], [900, 61], 8, 2, 64, 16, "bfloat16")]
    T = sum(news)
    k, v = (tensor(r.standard_normal((T, 2, 64)), "bfloat16")[0] for _ in range(2))
    c, d = cases
    # the free pages are those that the table holds for the new tokens already
    have = [n - m for n, m in zip(lens, news)]
    i32 = [ints(have), ints(news), ints(c["table"])]
    q, kp, vp = c["q"], c["kp"], c["vp"]
    grow = [-(-n // 16) > -(-h // 16) for n, h in zip(lens, have)]
    pool = ints([p for i, g in enumerate(grow) if g
                 for p in c["table"][i, -(-have[i] // 16):-(-lens[i] // 16)]] or [0])

    def step():
        st = O.pagedBlockTables(*i32, pool, 16, T)
        O.pagedCacheWrite(kp, vp, k, v, st.slots)
        return [O.pagedAttention(q, kp, vp, st.blockTable, st.starts, st.lens)]

    want = E.toHostF32(step()[0])
    d32 = [ints(d[n]) for n in ("table", "starts", "lens")]
    other = lambda: [O.pagedAttention(d["q"], d["kp"], d["vp"], *d32)]
    eager_d = lambda: E.toHostF32(other()[0])
    want_d = eager_d()
    first, second = _capture(step), _capture(other)
    for got in _replays(first, eager_d):
        np.testing.assert_array_equal(got[0], want)
    for _ in range(3):  # both in flight, one behind the other
        first[0]()
        second[0]()
        E.sync()
        np.testing.assert_array_equal(E.toHostF32(first[2][0]), want)
        np.testing.assert_array_equal(E.toHostF32(second[2][0]), want_d)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_captured_training_step(gpu, dtype):
    """Attention with its gradients captured, replayed between eager gradients of others."""
    r = np.random.default_rng(1)
    (q, _), (k, _), (v, _) = make(r, 400, 4, 2, 64, dtype)
    do, _ = tensor(r.standard_normal((400, 4, 64)), dtype)
    starts, others = ints([0, 33, 290, 400]), ints([0, 400])

    def step(s):
        out, stats = O.packedAttention(q, k, v, s, withLse=True)
        return [out, *O.packedAttentionGrad(q, k, v, s, out, stats, do)]

    want = [E.toHostF32(t) for t in step(starts)]
    eager = lambda: [E.toHostF32(t) for t in step(others)]
    want_e = eager()
    for got in _replays(_capture(lambda: step(starts)), eager):
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g, w)
    for g, w in zip(eager(), want_e):
        np.testing.assert_array_equal(g, w)


def test_training_step_descends_by_the_gradient(gpu):
    """The gradients of a packed attention inside a float64 loss: a step along them changes it
    as they say (the derivative along a direction, not how far it falls)."""
    r = np.random.default_rng(3)
    starts = [0, 40, 41, 170]
    x = [h for _, h in make(r, 170, 4, 2, 64, "float16")]
    w = r.standard_normal((170, 4, 64))
    do, doh = tensor(w, "float16")
    t = [tensor(h, "float16")[0] for h in x]
    out, stats = O.packedAttention(*t, ints(starts), withLse=True)
    grads = [E.toHostF32(g).astype(np.float64)
             for g in O.packedAttentionGrad(*t, ints(starts), out, stats, do)]
    _, bnd = R.packed_grad(*x, starts, doh, True, 64 ** -0.5, "float16")
    d = [r.standard_normal(h.shape) for h in x]
    eps = 1e-5
    loss = [(R.packed(*(h + s * eps * e for h, e in zip(x, d)), starts, True, 64 ** -0.5)[0]
             * doh).sum() for s in (1, -1)]
    along = (loss[0] - loss[1]) / (2 * eps)
    got = sum((g * e).sum() for g, e in zip(grads, d))
    bound = sum((b * np.abs(e)).sum() for b, e in zip(bnd, d))
    assert abs(got - along) <= bound + 1e-4 * abs(along)


def test_many_requests(gpu):
    """More requests than a wave has lanes, empty ones among them, in every kernel."""
    r = np.random.default_rng(5)
    news = [1, 0, 1, 2] * 40
    lens = [int(n) if m else int(n) * (i % 2) for i, (m, n) in
            enumerate(zip(news, r.integers(3, 200, 160)))]
    for width in (None, 300):
        c = paged_case(r, news, lens, 4, 2, 64, 16, "bfloat16", width=width)
        want, mag = paged_want(c, True, 0.125)
        check(paged_call(c), want, R.out_bound(want, mag, "bfloat16"))
    news = [1, 0, 40, 2] * 20
    lens = [n + int(m) for n, m in zip(news, r.integers(0, 200, 80))]
    c = paged_case(r, news, lens, 4, 2, 64, 16, "float16")
    want, mag = paged_want(c, True, 0.125)
    check(paged_call(c), want, R.out_bound(want, mag, "float16"))
    lens = list(r.integers(0, 30, 150))
    starts = np.concatenate([[0], np.cumsum(lens)])
    (q, qh), (k, kh), (v, vh) = make(r, starts[-1], 4, 2, 32, "bfloat16")
    for causal in (True, False):
        out, stats = O.packedAttention(q, k, v, ints(starts), causal=causal, withLse=True)
        want, _, mag = R.packed(qh, kh, vh, starts, causal, 32 ** -0.5)
        check(out, want, R.out_bound(want, mag, "bfloat16"))
        do, doh = tensor(r.standard_normal(qh.shape), "bfloat16")
        wants, bnds = R.packed_grad(qh, kh, vh, starts, doh, causal, 32 ** -0.5, "bfloat16")
        for g, w, b in zip(O.packedAttentionGrad(q, k, v, ints(starts), out, stats, do,
                                                 causal=causal), wants, bnds):
            check(g, w, b)
