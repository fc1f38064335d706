"""GPU checks of the packed and paged operators at the edges of their use: splits, hints, long
caches, replayed plans, single launches and the refusals of the library itself."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import _lib
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType, EagerError
from test_gpu_packed import DTYPES, check, ints, make, tensor
from test_gpu_paged import paged_call, paged_case, paged_want


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [2, 64])
def test_split_blocks(gpu, D, dtype, page):
    """Blocks of many key tiles, in several pieces, beside single tokens and short prompts."""
    news, lens = [40, 1, 33, 60], [3000, 2500, 33, 1800]
    c = paged_case(np.random.default_rng(D), news, lens, 4, 2, D, page, dtype)
    for causal in (True, False):
        want, mag = paged_want(c, causal, D ** -0.5)
        check(paged_call(c, causal=causal), want, R.out_bound(want, mag, dtype))


@pytest.mark.parametrize("news,lens", [([200, 1, 17], [900, 64, 17]), ([1, 1], [2500, 40])])
@pytest.mark.parametrize("width", [None, 400])
def test_any_hint_gives_the_result(gpu, news, lens, width):
    c = paged_case(np.random.default_rng(2), news, lens, 8, 2, 64, 16, "bfloat16", width=width)
    want, mag = paged_want(c, True, 0.125)
    for hint in (0, 1, 8, 9, 200, 2 ** 40):
        check(paged_call(c, maxNew=hint), want, R.out_bound(want, mag, "bfloat16"))


@pytest.mark.parametrize("H,Hkv,D", [(7, 7, 32), (40, 1, 64), (71, 1, 128), (15, 5, 64)])
def test_odd_groups(gpu, H, Hkv, D):
    """Groups that do not divide a block of rows, and ones larger than a decode block."""
    r = np.random.default_rng(H)
    starts = [0, 3, 3, 70]
    (q, qh), (k, kh), (v, vh) = make(r, 70, H, Hkv, D, "bfloat16")
    out, stats = O.packedAttention(q, k, v, ints(starts), withLse=True)
    want, _, mag = R.packed(qh, kh, vh, starts, True, D ** -0.5)
    check(out, want, R.out_bound(want, mag, "bfloat16"))
    do, doh = tensor(r.standard_normal(qh.shape), "bfloat16")
    for g, w, b in zip(O.packedAttentionGrad(q, k, v, ints(starts), out, stats, do),
                       *R.packed_grad(qh, kh, vh, starts, doh, True, D ** -0.5, "bfloat16")):
        check(g, w, b)
    for news, lens, width in (([1, 2], [300, 7], None), ([1, 2], [300, 7], 400),
                              ([60, 1], [90, 400], None)):
        c = paged_case(r, news, lens, H, Hkv, D, 8, "bfloat16", width=width)
        want, mag = paged_want(c, True, D ** -0.5)
        check(paged_call(c), want, R.out_bound(want, mag, "bfloat16"))


def test_cache_past_32_bit_offsets(gpu):
    """Pages behind 2^32 bytes (and 2^31 values) of the cache."""
    page, Hkv, D = 64, 4, 128
    pages = 2 ** 31 // (page * Hkv * D) + 600
    kp, vp = (E.empty(DType.BFLOAT16, (pages, Hkv, page, D)) for _ in range(2))
    r = np.random.default_rng(0)
    far = [pages - 1, 3, pages - 300, 2 ** 31 // (page * Hkv * D), 2 ** 30 // (page * Hkv * D)]
    n = 300
    slots = np.concatenate([p * page + np.arange(page) for p in far])[:n]
    (k, kh), (v, vh) = (tensor(r.standard_normal((n, Hkv, D)), "bfloat16") for _ in range(2))
    O.pagedCacheWrite(kp, vp, k, v, ints(slots))
    for news, width in ((1, 5), (1, 60), (40, 5)):
        q, qh = tensor(r.standard_normal((news, 8, D)), "bfloat16")
        table = np.full((1, width), -1)
        table[0, :5] = far
        got = O.pagedAttention(q, kp, vp, ints(table), ints([0, news]), ints([n]))
        want, _, _, mag = R.attend(qh, kh, vh, n - news, True, D ** -0.5)
        check(got, want, R.out_bound(want, mag, "bfloat16"))


def test_replayed_plans(gpu):
    """The same calls on new inputs (a recorded plan), attention as an intermediate."""
    r = np.random.default_rng(4)
    starts = ints([0, 30, 100])
    for _ in range(4):
        (q, qh), (k, kh), (v, vh) = make(r, 100, 4, 2, 64, "bfloat16")
        # doubled where nothing but the next op holds it
        got = O.add(*[O.packedAttention(q, k, v, starts)] * 2)
        want, _, mag = R.packed(qh, kh, vh, [0, 30, 100], True, 0.125)
        check(got, 2 * want, 2 * R.out_bound(want, mag, "bfloat16"))
        c = paged_case(r, [40, 1], [1900, 300], 8, 2, 64, 16, "bfloat16")
        got = O.add(*[paged_call(c)] * 2)
        want, mag = paged_want(c, True, 0.125)
        check(got, 2 * want, 2 * R.out_bound(want, mag, "bfloat16"))
        c = paged_case(r, [1, 1], [1900, 300], 8, 2, 64, 16, "bfloat16", width=300)
        got = O.add(*[paged_call(c)] * 2)
        want, mag = paged_want(c, True, 0.125)
        check(got, 2 * want, 2 * R.out_bound(want, mag, "bfloat16"))


def test_one_op_at_a_time(gpu):
    """MODE_OP_BY_OP gives the deferred results."""
    r = np.random.default_rng(8)
    (q, _), (k, _), (v, _) = make(r, 90, 4, 2, 64, "float16")
    do, _ = tensor(r.standard_normal((90, 4, 64)), "float16")
    c = paged_case(r, [1, 40], [300, 90], 4, 2, 64, 16, "float16")

    def run():
        out, stats = O.packedAttention(q, k, v, ints([0, 90]), withLse=True)
        t = [out, *O.packedAttentionGrad(q, k, v, ints([0, 90]), out, stats, do), paged_call(c),
             *O.pagedBlockTables(ints([3, 0]), ints([1, 4]), ints([[5, 0], [0, 0]]),
                                 ints([7, 2]), 4, 5)]
        return [E.toHostF32(x) if x.dtype != DType.INT32 else E.toHost(x) for x in t]

    want = run()
    E.setMode(E.MODE_OP_BY_OP)
    try:
        got = run()
    finally:
        E.setMode(E.MODE_DEFERRED)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)


def test_library_refusals(gpu):
    """What the library refuses by itself, the Python checks aside; nothing is launched."""
    def e(dt, *shape):
        return E.empty(dt, shape)

    b16, f32, i32 = DType.BFLOAT16, DType.FLOAT32, DType.INT32

    def refuse(match, op, operands, attrs):
        with pytest.raises((EagerError, O.TensorError), match=match):
            E.executeMi355xOp(op, operands, attrs)

    at = [("causal", "true"), ("scale", "0.0"), ("stats", "false")]
    starts = ints([0, 4])
    x = e(b16, 4, 2, 64)
    refuse("head", "packedAttention", [e(b16, 4, 2, 96)] * 3 + [starts], at)
    refuse("float", "packedAttention", [e(f32, 4, 2, 64)] * 3 + [starts], at)
    refuse("heads", "packedAttention", [e(b16, 4, 3, 64), x, x, starts], at)
    refuse("tokens", "packedAttention", [e(b16, 5, 2, 64), x, x, starts], at)
    refuse("int32", "packedAttention", [x, x, x, e(f32, 2)], at)
    refuse("starts", "packedAttention", [x, x, x, e(i32, 0)], at)
    refuse("scale", "packedAttention", [x] * 3 + [starts],
           [("causal", "true"), ("scale", "-1"), ("stats", "false")])
    pages = [e(b16, 3, 2, 16, 64) for _ in range(2)]
    at = [("causal", "true"), ("scale", "0.0"), ("max_new", "0")]
    table, lens = e(i32, 1, 3), e(i32, 1)
    refuse("requests", "pagedAttention", [x, *pages, table, e(i32, 3), lens], at)
    refuse("power of two", "pagedAttention", [x, *[e(b16, 3, 2, 12, 64)] * 2, table, starts,
                                              lens], at)
    refuse("2\\^30", "pagedAttention", [x, *pages, e(i32, 1, 2 ** 27), starts, lens], at)
    refuse("max_new", "pagedAttention", [x, *pages, table, starts, lens],
           at[:2] + [("max_new", "-1")])
    k, slots = e(b16, 4, 2, 64), ints([0, 1, 2, 3])
    refuse("one tensor", "pagedCacheWrite", [pages[0], pages[0], k, k, slots], [])
    fixed = E.fromHost(np.zeros((3, 2, 16, 64), np.float32), b16)
    refuse("immutable", "pagedCacheWrite", [fixed, pages[1], k, k, slots], [])
    refuse("immutable", "pagedCacheWrite", [pages[0], O.add(fixed, fixed), k, k, slots], [])
    refuse("slots", "pagedCacheWrite", [*pages, k, k, ints([0])], [])
    refuse("do not fit", "pagedCacheWrite", [*pages, e(b16, 4, 1, 64), e(b16, 4, 1, 64), slots],
           [])
    i2, tab = ints([1, 1]), e(i32, 2, 3)
    refuse("page", "pagedBlockTables", [i2, i2, tab, i2], [("page_size", "3"), ("tokens", "2")])
    refuse("tokens", "pagedBlockTables", [i2, i2, tab, i2],
           [("page_size", "4"), ("tokens", "-2")])
    refuse("eager", "pagedBlockTables", [ints([1]), i2, tab, i2],
           [("page_size", "4"), ("tokens", "2")])


def test_write_beside_a_view(gpu):
    """Pages that another tensor shares are not changed under it."""
    pages = [E.empty(DType.BFLOAT16, (2, 1, 4, 32)) for _ in range(2)]
    row, slot = E.empty(DType.BFLOAT16, (1, 1, 32)), ints([5])
    for p in pages:
        view = O.reshape(p, [8, 1, 32])
        with pytest.raises(EagerError, match="shares its memory"):
            O.pagedCacheWrite(*pages, row, row, slot)
        del view
    O.pagedCacheWrite(*pages, row, row, slot)


def test_operands_that_are_views(gpu):
    """Transposed, sliced, broadcast and computed operands, not yet materialized."""
    r = np.random.default_rng(12)
    T, H, D = 77, 4, 64
    x, xh = tensor(r.standard_normal((H, T, D)), "bfloat16")
    y, yh = tensor(r.standard_normal((T + 9, 2, 2 * D)), "bfloat16")
    z, zh = tensor(r.standard_normal((T, D)), "bfloat16")
    qh, kh = xh.transpose(1, 0, 2), yh[4:4 + T, :, D:]
    vh = np.repeat(zh[:, None], 2, axis=1)
    starts = [0, 20, 77]

    def operands():
        return (O.transpose(x, [1, 0, 2]),
                O.slice_(y, [4, 0, D], [4 + T, 2, 2 * D], [1, 1, 1]),
                O.broadcastTo(z, [T, 2, D], [0, 2]))

    out, stats = O.packedAttention(*operands(), ints(starts), withLse=True)
    want, _, mag = R.packed(qh, kh, vh, starts, True, D ** -0.5)
    check(out, want, R.out_bound(want, mag, "bfloat16"))
    one = O.broadcastTo(E.fromHost(np.float32(1.0).reshape(1), DType.BFLOAT16), [T, H, D], [0])
    got = O.packedAttentionGrad(*operands(), ints(starts), out, stats, one)
    for g, w, b in zip(got, *R.packed_grad(qh, kh, vh, starts, np.ones((T, H, D)), True,
                                           D ** -0.5, "bfloat16")):
        check(g, w, b)
    page = 4
    kp, vp = (E.empty(DType.BFLOAT16, (20, 2, page, D)) for _ in range(2))
    _, k, v = operands()
    O.pagedCacheWrite(kp, vp, k, v, O.iota(DType.INT32, [T], 0))
    table = O.reshape(O.iota(DType.INT32, [20], 0), [1, 20])
    check(O.pagedAttention(operands()[0], kp, vp, table, ints([0, T]), ints([T])),
          *[f(*R.packed(qh, kh, vh, [0, T], True, D ** -0.5)[::2]) for f in
            (lambda w, m: w, lambda w, m: R.out_bound(w, m, "bfloat16"))])


@pytest.mark.parametrize("news", [[3, 0], [50, 2]])
def test_nothing_to_attend(gpu, news):
    """No requests, tables of no width, a cache of no pages, a free list of none."""
    r = np.random.default_rng(1)
    T = sum(news)
    q, _ = tensor(r.standard_normal((T, 4, 64)), "bfloat16")
    starts, lens = ints(np.concatenate([[0], np.cumsum(news)])), ints([60, 2])
    kp, vp = (E.empty(DType.BFLOAT16, (3, 2, 16, 64)) for _ in range(2))
    no_pages = [E.empty(DType.BFLOAT16, (0, 2, 16, 64)) for _ in range(2)]
    for args in ((kp, vp, E.empty(DType.INT32, (0, 4)), ints([0]), E.empty(DType.INT32, (0,))),
                 (kp, vp, E.empty(DType.INT32, (2, 0)), starts, lens),
                 (*no_pages, ints([[0, 1, 2, 3], [2, 1, 0, 0]]), starts, lens)):
        assert not E.toHostF32(O.pagedAttention(q, *args)).any()
    k, _ = tensor(r.standard_normal((T, 2, 64)), "bfloat16")
    O.pagedCacheWrite(*no_pages, k, k, O.iota(DType.INT32, [T], 0))
    for table, pool in ((np.zeros((2, 0)), [4, 5]), (np.zeros((2, 4)), []),
                        (np.zeros((2, 4)), [2 ** 27, -3, 2 ** 31 - 1, 2 ** 28, 1])):
        got = O.pagedBlockTables(ints([0, 0]), ints(news), ints(table), ints(pool), 16, T)
        for g, w in zip(got, R.block_tables([0, 0], news, table.astype(np.int64), pool, 16, T)):
            np.testing.assert_array_equal(E.toHost(g), w)


def test_write_through_the_c_interface(gpu):
    """No room for outputs is needed, and tensors of another context are refused."""
    lib = _lib.load()
    kp, vp = (E.empty(DType.BFLOAT16, (2, 1, 4, 32)) for _ in range(2))
    row, want = tensor(np.random.default_rng(0).standard_normal((1, 1, 32)), "bfloat16")
    slot, n = ints([6]), C.c_int(9)

    def call(ctx, operands):
        ops = (C.c_void_p * 5)(*operands)
        return lib.rew_mi355x_execute(ctx, b"pagedCacheWrite", ops, 5, None, None, 0, None, 0,
                                      C.byref(n))

    mine = [t.handle for t in (kp, vp, row, row, slot)]
    assert call(E.context(), mine) == 0 and n.value == 0
    for p in (kp, vp):
        np.testing.assert_array_equal(E.toHostF32(p)[1, 0, 2], want[0, 0])
    other, shape, far = C.c_void_p(), (C.c_int64 * 4)(2, 1, 4, 32), C.c_void_p()
    assert lib.rew_mi355x_init(0, C.byref(other)) == 0
    if other.value == C.cast(E.context(), C.c_void_p).value:
        return  # (contexts of a device are shared)
    assert lib.rew_mi355x_alloc(other, int(DType.BFLOAT16), shape, 4, C.byref(far)) == 0
    assert call(E.context(), [far.value, *mine[1:]]) != 0
    assert b"cross-device" in lib.rew_mi355x_last_error()
    lib.rew_mi355x_release(far)
