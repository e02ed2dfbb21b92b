"""Plain 64-bit forms of the serving operators (numpy), for the tests."""
import numpy as np


def plan(lens, new, page, free, cursor, table, n_slots):
    """(code, table, slots, cu, cursor, pages taken) of wg_kv_plan."""
    table = table.copy()
    R = len(lens)
    bad = (-1 * np.ones(n_slots, np.int32), np.zeros(R + 1, np.int32))
    code = 0
    for n, m in zip(lens, new):
        if n < 0 or m < 0 or m > n:
            code = max(code, 1)
        elif -(-n // page) > table.shape[1]:
            code = max(code, 2)
    ok = [(int(n), int(m)) for n, m in zip(lens, new) if not (n < 0 or m < 0 or m > n)]
    if sum(m for _, m in ok) > n_slots:
        code = max(code, 3)
    take = sum(-(-n // page) + -(-(n - m) // page) * -1 for n, m in ok)
    if cursor < 0 or cursor + take > len(free):
        code = max(code, 4)
    if code:
        return (code, table) + bad + (cursor, 0)
    slots, cu, at = [], [0], cursor
    for r, (n, m) in enumerate(ok):
        for c in range(-(-(n - m) // page), -(-n // page)):
            table[r, c] = free[at]
            at += 1
        for pos in range(n - m, n):
            slots.append(table[r, pos // page] * page + pos % page)
        cu.append(len(slots))
    out = -np.ones(n_slots, np.int64)
    out[:len(slots)] = slots
    return 0, table, out.astype(np.int32), np.array(cu, np.int32), at, at - cursor


def needed_scale(amax):
    """The least 2^e (e >= -126) with amax <= 127 * 2^e; 0 for 0."""
    if amax == 0:
        return 0.0
    e = int(np.floor(np.log2(float(amax)))) - 8
    while 127.0 * 2.0 ** e < amax:
        e += 1
    return 2.0 ** max(e, -126)


def append(codes, scales, k, v, slots):
    """wg_kv8_append in place on numpy codes and scales; k, v float64 [n, H, D]."""
    num, _, H, page, _ = codes.shape
    t = 0
    while t < len(slots):
        s = int(slots[t])
        if s < 0 or s >= num * page:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == s + n and (s + n) % page:
            n += 1
        pg, first = s // page, s % page
        for j, x in enumerate((k, v)):
            for h in range(H):
                y = x[t:t + n, h]
                mag = np.abs(y[np.isfinite(y)])
                need = needed_scale(mag.max() if mag.size else 0.0)
                old = float(scales[pg, j, h]) if first else 0.0
                new = max(old, need)
                if first and new > old > 0:
                    codes[pg, j, h, :first] = np.rint(codes[pg, j, h, :first] * (old / new))
                with np.errstate(invalid="ignore", divide="ignore"):
                    q = y / new if new > 0 else np.zeros_like(y)
                q = np.where(np.isnan(y), 0.0, q)
                codes[pg, j, h, first:first + n] = np.rint(np.clip(q, -127, 127))
                scales[pg, j, h] = new
        t += n


def attention(codes, scales, q, cu, lens, table, n_head, causal, scale, max_q=None):
    """{row: [n_head, D] float64} of wg_kv8_attention, and the largest |v| each row and head sees.
    codes and scales: numpy, or anything indexable by (page, j, head) giving numpy blocks."""
    num, _, H, page, D = codes.shape
    G = n_head // H
    out, most = {}, {}
    for r in range(len(lens)):
        a, b = int(cu[r]), int(cu[r + 1])
        if a < 0 or b < a or b > q.shape[0]:
            continue
        n = max(0, min(int(lens[r]), table.shape[1] * page))
        ids = [int(table[r, c]) for c in range(-(-n // page))]
        kv = np.zeros((2, H, len(ids) * page, D))
        ok = np.zeros(len(ids) * page, bool)
        for i, pg in enumerate(ids):
            if 0 <= pg < num:
                ok[i * page:(i + 1) * page] = True
                kv[:, :, i * page:(i + 1) * page] = (codes[pg].astype(np.float64) *
                                                     scales[pg].astype(np.float64)[..., None, None])
        for i in range(b - a):
            if max_q is not None and i >= max_q:
                continue
            seen = n - (b - a) + i + 1 if causal else n
            vis = np.flatnonzero(ok[:max(0, min(seen, n))])
            o, mv = np.zeros((n_head, D)), np.zeros((n_head, 1))
            for h in range(n_head):
                if vis.size:
                    kk, vv = kv[0, h // G][vis], kv[1, h // G][vis]
                    s = scale * (kk @ q[a + i, h].astype(np.float64))
                    w = np.exp(s - s.max())
                    o[h] = (w / w.sum()) @ vv
                    mv[h] = np.abs(vv).max()
            out[a + i], most[a + i] = o, mv
    return out, most


def sample(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """(token, log-prob) of wg_sample_rows for one row, x float64."""
    x = np.where(np.isnan(x), -np.inf, x)
    mx = x.max()
    if mx == -np.inf:
        return -1, -np.inf
    t = T if T > 0 else 1.0
    with np.errstate(invalid="ignore"):
        z = np.where(x == mx, 0.0, (x - mx) / t)
    w = np.exp(z)
    logz = np.log(w.sum())
    order = np.argsort(-x, kind="stable")
    if not T > 0:
        return int(order[0]), -logz
    n = k if 0 < k < x.size else x.size
    ws = w[order[:n]]
    if not p >= 1:
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        n = max(1, int((before < p * ws.sum()).sum()))
    n = max(1, min(n, int((w[order] >= m).sum())))
    kept = np.sort(order[:n])
    cum = np.cumsum(w[kept])
    tok = int(kept[min(n - 1, int((cum <= u * cum[-1]).sum()))])
    return tok, z[tok] - logz
