"""Plain float64 forms of the packed and paged operators, and error bounds for the kernels.

Every bound counts roundings: h is half a step of the operands' dtype (bfloat16 2^-8, float16
2^-11), the error of one rounding relative to the value.  The kernels round the
probabilities (and dS) once to that dtype for the second product and each result once; scores,
softmax statistics and sums are float32, whose error is taken as F32 of the sums of absolute
values: 128 products of a score lose at most 128 * 2^-24 = 8e-6 of sum |q||k| (below 30
here after the scale, so 2.3e-4 of a probability at the most, far less on average), and exp2,
the sums and the normalisation a few 2^-24 more.
"""
import numpy as np

F32 = 3e-4
HALF = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def scores(q, k, scale):
    """[H, n, L] scores of q [n, H, D] over k [L, Hkv, D] in float64."""
    g = q.shape[1] // k.shape[1]
    kk = np.repeat(k, g, axis=1)
    return np.matmul(q.transpose(1, 0, 2), kk.transpose(1, 2, 0)) * scale


def attend(q, k, v, first, causal, scale, there=None):
    """(out [n, H, D], lse [n, H], p [H, n, L], bound [n, H, D]) of one sequence whose
    query i is at position first + i; `there`: which keys exist."""
    n, L = q.shape[0], k.shape[0]
    s = scores(q, k, scale)
    seen = np.ones((n, L), bool)
    if causal:
        seen = np.arange(L)[None, :] <= first + np.arange(n)[:, None]
    if there is not None:
        seen = seen & there[None, :]
    s = np.where(seen[None], s, -np.inf)
    m = s.max(2, keepdims=True, initial=-np.inf)
    e = np.exp(s - np.where(np.isinf(m), 0.0, m))
    total = e.sum(2, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (np.where(np.isinf(m), 0.0, m) + np.log(total))[..., 0]
    p = e / np.where(total == 0, 1.0, total)
    # a key that no query sees does not take part, whatever its value
    used = seen.any(0)
    vv = np.repeat(np.where(used[:, None, None], v, 0.0), q.shape[1] // k.shape[1], axis=1)
    vv = vv.transpose(1, 0, 2)
    return (np.matmul(p, vv).transpose(1, 0, 2), lse.T, p,
            np.matmul(p, np.abs(vv)).transpose(1, 0, 2))


def packed(q, k, v, starts, causal, scale):
    """out, lse and the bound's sum p |v| over all sequences; zeros elsewhere."""
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    mag = np.zeros(q.shape)
    for a, b in zip(starts[:-1], starts[1:]):
        if b > a:
            out[a:b], lse[a:b], _, mag[a:b] = attend(q[a:b], k[a:b], v[a:b], 0, causal, scale)
    return out, lse, mag


def out_bound(out, mag, dtype):
    h = HALF[dtype]
    return (h + F32) * mag + h * np.abs(out) + 1e-7


def packed_grad(q, k, v, starts, do, causal, scale, dtype):
    """(dq, dk, dv) and their bounds."""
    h = HALF[dtype]
    g = q.shape[1] // k.shape[1]
    res = [np.zeros(q.shape), np.zeros(k.shape), np.zeros(k.shape)]
    bnd = [np.zeros(q.shape), np.zeros(k.shape), np.zeros(k.shape)]
    for a, b in zip(starts[:-1], starts[1:]):
        if b <= a:
            continue
        n = b - a
        out, _, p, _ = attend(q[a:b], k[a:b], v[a:b], 0, causal, scale)
        qh, dh, oh = (x.transpose(1, 0, 2) for x in (q[a:b], do[a:b], out))
        kh = np.repeat(k[a:b], g, axis=1).transpose(1, 0, 2)
        vh = np.repeat(v[a:b], g, axis=1).transpose(1, 0, 2)
        dp = np.matmul(dh, vh.transpose(0, 2, 1))
        delta = (dh * oh).sum(2, keepdims=True)
        ds = p * (dp - delta)
        # dS: one rounding, half a step of the rest that delta adds to out (of the row's
        # largest value), float32 sums
        mag_dp = np.matmul(np.abs(dh), np.abs(vh).transpose(0, 2, 1))
        mag_delta = (np.abs(dh) * np.abs(oh)).sum(2, keepdims=True)
        e_rest = h / 254 * np.abs(dh).sum(2, keepdims=True) * np.abs(oh).max(2, keepdims=True)
        e_ds = h * np.abs(ds) + p * (1.1 * e_rest + F32 * (mag_dp + mag_delta))
        e_p = (h + F32) * p

        def group(x):  # [H, n, D] -> [n, Hkv, D], summed over each group
            return x.reshape(-1, g, n, x.shape[2]).sum(1).transpose(1, 0, 2)

        res[0][a:b] = (np.matmul(ds, kh) * scale).transpose(1, 0, 2)
        bnd[0][a:b] = (np.matmul(e_ds, np.abs(kh)) * scale).transpose(1, 0, 2)
        res[1][a:b] = group(np.matmul(ds.transpose(0, 2, 1), qh) * scale)
        bnd[1][a:b] = group(np.matmul(e_ds.transpose(0, 2, 1), np.abs(qh)) * scale)
        res[2][a:b] = group(np.matmul(p.transpose(0, 2, 1), dh))
        bnd[2][a:b] = group(np.matmul(e_p.transpose(0, 2, 1), np.abs(dh)))
    return res, [e + h * np.abs(r) + 1e-7 for e, r in zip(bnd, res)]


def gather_pages(pages, table, n):
    """([n, Hkv, D] rows of one request, which of them exist)."""
    ps = pages.shape[2]
    rows = np.zeros((n, pages.shape[1], pages.shape[3]))
    there = np.zeros(n, bool)
    for j in range(n):
        b = j // ps
        if b < len(table) and 0 <= table[b] < pages.shape[0]:
            rows[j], there[j] = pages[table[b], :, j % ps], True
    return rows, there


def block_tables(cached, new, table, free, page, tokens):
    """pagedBlockTables one request and token at a time."""
    table = np.array(table)
    out = np.full(table.shape, -1, np.int64)
    slots, positions = np.full(tokens, -1, np.int64), np.zeros(tokens, np.int64)
    starts, lens, t, taken = [], [], 0, 0
    for r in range(len(cached)):
        c, f = max(int(cached[r]), 0), max(int(new[r]), 0)
        have, want = -(-c // page), -(-(c + f) // page)
        row = {}
        for j in range(want):
            if j >= have:
                row[j] = int(free[taken]) if taken < len(free) else -1
                taken += 1
            else:
                row[j] = int(table[r, j]) if j < table.shape[1] else -1
        for j in range(min(want, table.shape[1])):
            out[r, j] = row[j]
        starts.append(min(t, tokens))
        for p in range(c, c + f):
            if t < tokens:
                e = row[p // page] if p // page < table.shape[1] else -1
                slots[t] = e * page + p % page if 0 <= e * page + p % page < 2 ** 31 else -1
                positions[t] = p
            t += 1
        lens.append(c + f)
    return out, slots, positions, np.array(starts + [min(t, tokens)]), np.array(lens), \
        np.array([taken])
