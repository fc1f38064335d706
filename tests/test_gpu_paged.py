"""GPU checks of the paged cache: block tables, writes in place, attention over the pages."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import packed_ref as R
from rew_amd import eager as E
from rew_amd import ops as O
from rew_amd.eager import DType
from test_gpu_packed import DTYPES, check, ints, tensor


@pytest.mark.parametrize("page", [1, 16, 64, 256])
@pytest.mark.parametrize("cached,new", [
    ([0], [1]), ([5], [0]), ([15, 16, 17], [1, 1, 1]), ([0, 0, 100, 7], [300, 0, 1, 57]),
    (list(range(70)), [1] * 70), ([3, -2, 9], [2, 4, -7]), ([250] * 300, [1, 0, 9] * 100)])
def test_block_tables(gpu, page, cached, new):
    r = np.random.default_rng(len(cached) + page)
    width = max(-(-(max(c, 0) + max(n, 0)) // page) for c, n in zip(cached, new)) + 2
    need = sum(-(-(max(c, 0) + max(n, 0)) // page) + -(-max(c, 0) // page)
               for c, n in zip(cached, new))
    order = r.permutation(need + 9)
    table = np.full((len(cached), width), -1, np.int64)
    at = 0
    for i, c in enumerate(cached):
        have = -(-max(c, 0) // page)
        table[i, :have] = order[at:at + have]
        at += have
    table[0, width - 1] = 77  # whatever lies behind a request's pages is not kept
    free, total = order[at:], sum(max(n, 0) for n in new)
    for tokens, pool in ((total, free), (total + 5, free), (max(total - 1, 0), free),
                         (total, free[:1])):
        got = O.pagedBlockTables(ints(cached), ints(new), ints(table), ints(pool), page, tokens)
        want = R.block_tables(cached, new, table, pool, page, tokens)
        for name, g, w in zip("table slots positions starts lens taken".split(), got, want):
            np.testing.assert_array_equal(E.toHost(g), w, err_msg=name)


def test_block_tables_too_narrow(gpu):
    """Tokens past the table's width get no slot."""
    got = O.pagedBlockTables(ints([6]), ints([9]), ints([[4, 2, 9]]), ints([7, 8, 1]), 4, 9)
    want = R.block_tables([6], [9], [[4, 2, 9]], [7, 8, 1], 4, 9)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(E.toHost(g), w)
    assert (E.toHost(got[1])[6:] == -1).all()


def test_block_tables_of_nothing(gpu):
    got = O.pagedBlockTables(E.empty(DType.INT32, (0,)), E.empty(DType.INT32, (0,)),
                             E.empty(DType.INT32, (0, 4)), ints([3]), 16, 2)
    np.testing.assert_array_equal(E.toHost(got[1]), [-1, -1])
    np.testing.assert_array_equal(E.toHost(got[3]), [0])
    np.testing.assert_array_equal(E.toHost(got[5]), [0])


def new_pages(r, pages, Hkv, page, D, dtype):
    """Pages with values in every row, as (tensor, float64 values), filled by the op itself."""
    shape = (pages, Hkv, page, D)
    kp, vp = E.empty(DTYPES[dtype], shape), E.empty(DTYPES[dtype], shape)
    n = pages * page
    k, kh = tensor(r.standard_normal((n, Hkv, D)), dtype)
    v, vh = tensor(r.standard_normal((n, Hkv, D)), dtype)
    O.pagedCacheWrite(kp, vp, k, v, ints(np.arange(n)))
    as_pages = [x.reshape(pages, page, Hkv, D).transpose(0, 2, 1, 3).copy() for x in (kh, vh)]
    return kp, vp, *as_pages


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hkv,D,page", [(1, 32, 1), (3, 64, 16), (8, 128, 32), (2, 8, 4)])
def test_cache_write(gpu, dtype, Hkv, D, page):
    r = np.random.default_rng(D + page)
    kp, vp, kh, vh = new_pages(r, 20, Hkv, page, D, dtype)
    np.testing.assert_array_equal(E.toHostF32(kp), kh)
    np.testing.assert_array_equal(E.toHostF32(vp), vh)
    slots = r.permutation(20 * page)[:13]
    slots[[2, 5, 7]] = [-1, 20 * page, 2 ** 31 - 1]  # nothing is written for these
    (k, kn), (v, vn) = (tensor(r.standard_normal((len(slots), Hkv, D)), dtype) for _ in range(2))
    old = O.add(kp, kp)  # recorded before the write: it reads the old rows
    O.pagedCacheWrite(kp, vp, k, v, ints(slots))
    new = O.add(kp, kp)
    np.testing.assert_array_equal(E.toHostF32(old), 2 * kh)
    for t, s in enumerate(slots):
        if 0 <= s < 20 * page:
            kh[s // page, :, s % page], vh[s // page, :, s % page] = kn[t], vn[t]
    np.testing.assert_array_equal(E.toHostF32(kp), kh)
    np.testing.assert_array_equal(E.toHostF32(vp), vh)
    np.testing.assert_array_equal(E.toHostF32(new), 2 * kh)


def test_cache_write_of_nothing(gpu):
    kp, vp, kh, _ = new_pages(np.random.default_rng(0), 2, 1, 2, 32, "bfloat16")
    none = E.empty(DType.BFLOAT16, (0, 1, 32))
    O.pagedCacheWrite(kp, vp, none, none, E.empty(DType.INT32, (0,)))
    np.testing.assert_array_equal(E.toHostF32(kp), kh)


def paged_case(r, news, lens, H, Hkv, D, page, dtype, pages=None, width=None):
    """Random pages and tables for requests of `lens` keys and `news` new tokens."""
    blocks = [-(-max(n, 0) // page) for n in lens]
    pages = pages or sum(blocks) + 3
    width = max(blocks) + 1 if width is None else width
    kp, vp, kh, vh = new_pages(r, pages, Hkv, page, D, dtype)
    order = r.permutation(pages)
    table = np.full((len(lens), width), -1, np.int64)
    at = 0
    for i, b in enumerate(blocks):
        table[i, :b] = order[at:at + b][:width]
        at += b
    starts = np.concatenate([[0], np.cumsum(news)])
    q, qh = tensor(r.standard_normal((starts[-1], H, D)) * 1.5, dtype)
    return dict(q=q, kp=kp, vp=vp, qh=qh, kh=kh, vh=vh, table=table, starts=starts, lens=lens)


def paged_want(c, causal, scale):
    want, mag = np.zeros(c["qh"].shape), np.zeros(c["qh"].shape)
    for i, n in enumerate(c["lens"]):
        a, b = c["starts"][i], c["starts"][i + 1]
        if b == a:
            continue
        k, there = R.gather_pages(c["kh"], c["table"][i], max(n, 0))
        v, _ = R.gather_pages(c["vh"], c["table"][i], max(n, 0))
        want[a:b], _, _, mag[a:b] = R.attend(c["qh"][a:b], k, v, n - (b - a), causal, scale, there)
    return want, mag


def paged_call(c, **kw):
    return O.pagedAttention(c["q"], c["kp"], c["vp"], ints(c["table"]), ints(c["starts"]),
                            ints(c["lens"]), **kw)


STEPS = {  # new tokens, keys (the new ones among them)
    "first": ([1], [1]), "decode": ([1, 1, 1], [64, 65, 700]), "late": ([1], [3000]),
    "many": ([1] * 40, list(range(1, 400, 10))), "verify": ([4, 1, 3], [200, 30, 129]),
    "mixed": ([1, 90, 0, 1, 33], [300, 90, 50, 1, 433]), "chunk": ([200], [600]),
    "chunk_only": ([130, 70], [130, 70]),
}


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("H,Hkv,D,page", [(4, 4, 32, 1), (8, 2, 64, 16), (8, 1, 128, 32),
                                          (6, 2, 128, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention(gpu, step, H, Hkv, D, page, dtype):
    news, lens = STEPS[step]
    r = np.random.default_rng(sum(lens) + D + page)
    c = paged_case(r, news, lens, H, Hkv, D, page, dtype)
    want, mag = paged_want(c, True, D ** -0.5)
    check(paged_call(c), want, R.out_bound(want, mag, dtype))
    check(paged_call(c, maxNew=max(news)), want, R.out_bound(want, mag, dtype))


@pytest.mark.parametrize("step", ["first", "decode", "many", "verify"])
@pytest.mark.parametrize("H,Hkv,D,page", [(4, 4, 32, 1), (8, 2, 64, 16), (6, 2, 128, 128)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_wide_tables(gpu, step, H, Hkv, D, page, dtype):
    """A table with room for many more keys chooses other kernels."""
    news, lens = STEPS[step]
    r = np.random.default_rng(sum(lens) + D + page)
    c = paged_case(r, news, lens, H, Hkv, D, page, dtype, width=5000 // page)
    want, mag = paged_want(c, True, D ** -0.5)
    check(paged_call(c), want, R.out_bound(want, mag, dtype))


@pytest.mark.parametrize("step", ["decode", "mixed"])
def test_paged_attention_all_keys_and_scale(gpu, step):
    news, lens = STEPS[step]
    c = paged_case(np.random.default_rng(7), news, lens, 8, 2, 64, 16, "bfloat16")
    want, mag = paged_want(c, False, 0.3)
    check(paged_call(c, causal=False, scale=0.3), want, R.out_bound(want, mag, "bfloat16"))


@pytest.mark.parametrize("page", [1, 16, 64])
def test_paged_attention_missing_pages(gpu, page):
    """Keys whose page is absent, out of range or past the table are not seen; rows at
    negative positions and rows of no request give zeros."""
    r = np.random.default_rng(page)
    news, lens = [1, 3, 70, 9, 2], [500, 333, 200, 4, 0]
    c = paged_case(r, news, lens, 4, 2, 64, page, "bfloat16")
    n = c["kp"].shape[0]
    for row, col, v in ((0, 0, -1), (0, 3, n), (1, 1, -7), (2, 0, 2 ** 31 - 1), (2, 2, -1)):
        if col < c["table"].shape[1]:
            c["table"][row, col] = v
    c["lens"] = [500, 333, 200, 4, -5]
    want, mag = paged_want(c, True, 0.125)
    assert not want[c["starts"][3]:c["starts"][3] + 5].any() and not want[-2:].any()
    check(paged_call(c), want, R.out_bound(want, mag, "bfloat16"))
    c["table"][:] = -1
    assert not E.toHostF32(paged_call(c)).any()


def test_paged_attention_rows_behind_the_last_request(gpu):
    c = paged_case(np.random.default_rng(1), [2, 1], [40, 9], 4, 2, 64, 16, "float16")
    c["q"], c["qh"] = tensor(np.random.default_rng(2).standard_normal((50, 4, 64)), "float16")
    want, mag = paged_want(c, True, 0.125)
    check(paged_call(c), want, R.out_bound(want, mag, "float16"))


def test_paged_attention_unused_rows_may_hold_anything(gpu):
    """NaN and infinity in pages of others, and behind the last key of a page."""
    r = np.random.default_rng(6)
    for news, lens in (([1, 1], [37, 100]), ([40, 1], [77, 5])):
        c = paged_case(r, news, lens, 8, 2, 64, 16, "bfloat16")
        used = np.zeros((c["kp"].shape[0], 16), bool)
        for i, n in enumerate(lens):
            for j in range(n):
                used[c["table"][i, j // 16], j % 16] = True
        bad = np.flatnonzero(~used.reshape(-1))
        x = np.full((len(bad), 2, 64), np.nan)
        x[::2] = np.inf
        t, _ = tensor(x, "bfloat16")
        O.pagedCacheWrite(c["kp"], c["vp"], t, t, ints(bad))
        want, mag = paged_want(c, True, 0.125)
        check(paged_call(c), want, R.out_bound(want, mag, "bfloat16"))


def test_paged_equals_packed_prompt(gpu):
    """A prompt written into pages and read back attends like the packed prompt itself."""
    r = np.random.default_rng(9)
    lens, page = [100, 1, 250], 16
    starts = np.concatenate([[0], np.cumsum(lens)])
    (q, qh), (k, kh), (v, vh) = (tensor(r.standard_normal((351, h, 128)), "bfloat16")
                                 for h in (8, 2, 2))
    free = r.permutation(40)
    table = np.full((3, 20), -1)
    bt, slots, pos, st, ln, taken = O.pagedBlockTables(ints([0, 0, 0]), ints(lens), ints(table),
                                                       ints(free), page, 351)
    np.testing.assert_array_equal(E.toHost(st), starts)
    assert E.toHost(taken)[0] == 7 + 1 + 16
    shape = (40, 2, page, 128)
    kp, vp = E.empty(DType.BFLOAT16, shape), E.empty(DType.BFLOAT16, shape)
    O.pagedCacheWrite(kp, vp, k, v, slots)
    paged = O.pagedAttention(q, kp, vp, bt, st, ln)
    want, _, mag = R.packed(qh, kh, vh, starts, True, 128 ** -0.5)
    check(paged, want, R.out_bound(want, mag, "bfloat16"))
    check(O.packedAttention(q, k, v, st), want, R.out_bound(want, mag, "bfloat16"))
