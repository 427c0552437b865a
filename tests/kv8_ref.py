"""Plain 64-bit statements of the 8-bit paged KV cache's operators and of
sm_draw (numpy), for the tests. E4M3 rounding is written out here."""
import numpy as np

PAGE = 32
TOP = {"e4m3": 448.0, "i8": 127.0}


def e4m3_table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m / 8 * 2.0**-6, (1 + m / 8) * 2.0 ** (e - 7.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c & 128, -v, v)


E4M3 = e4m3_table()


def decode(codes, fmt):
    return E4M3[codes] if fmt == "e4m3" else codes.view(np.int8).astype(np.float64)


def encode(x, fmt):
    """The nearest code, ties to the even one (x within the type's range)."""
    if fmt == "i8":
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    e = np.floor(np.log2(np.maximum(a, 2.0**-30)))
    e = np.where(2.0 ** (e + 1) <= a, e + 1, np.where(2.0**e > a, e - 1, e))
    step = 2.0 ** (np.maximum(e, -6) - 3)
    v = np.rint(a / step) * step
    pos = E4M3[:127]
    code = np.searchsorted(pos, v)
    assert np.all(pos[code] == v)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def page_scale(top, fmt):
    """The smallest power of two s, 2^-100 at least, with top <= TOP s."""
    top = np.asarray(top, np.float64)
    out = np.full(top.shape, 2.0**-100)
    while True:
        low = top > TOP[fmt] * out
        if not low.any():
            return out
        jump = np.where(top > TOP[fmt] * out * 2.0**10, 2.0**10, 2.0)
        out = np.where(low, out * jump, out)


def append(codes, scales, k, v, slots, fmt):
    """codes [P, H, 2, 32, D] and scales [P, H, 2] after the call."""
    codes, scales = codes.copy(), scales.astype(np.float64)
    n_slots = codes.shape[0] * PAGE
    i = 0
    while i < len(slots):
        if not 0 <= slots[i] < n_slots:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % PAGE:
            j += 1
        page, a = divmod(int(slots[i]), PAGE)
        for w, x in enumerate((k, v)):
            for h in range(codes.shape[1]):
                r = x[i:j, h].astype(np.float64)
                old = scales[page, h, w] if a else 0.0
                if not np.isfinite(r).all() or np.isnan(old):
                    scales[page, h, w] = np.nan
                    codes[page, h, w, a:a + j - i] = 0
                    continue
                s = max(old, float(page_scale(np.abs(r).max(), fmt)))
                if a and s > old:
                    codes[page, h, w, :a] = encode(decode(codes[page, h, w, :a], fmt) * (old / s), fmt)
                codes[page, h, w, a:a + j - i] = encode(r / s, fmt)
                scales[page, h, w] = s
        i = j
    return codes, scales


def attend(codes, scales, fmt, q, lens, first, table, scale, window=0):
    """(out, error scale): rows of no sequence are NaN; the second is
    sum p |v| / sum p of every element, what rounding errors scale with."""
    P, H, _, _, D = codes.shape
    T, Hq, _ = q.shape
    G = Hq // H
    out = np.full((T, Hq, D), np.nan)
    mag = np.ones((T, Hq, D))
    for s in range(len(lens)):
        n = first[s + 1] - first[s]
        for i in range(n):
            pos = lens[s] - n + i
            lo = max(0, pos - window + 1) if window else 0
            js = [j for j in range(lo, pos + 1) if j // PAGE < table.shape[1] and 0 <= table[s, j // PAGE] < P]
            row = first[s] + i
            if not js:
                out[row] = 0
                continue
            pg, of = table[s, np.array(js) // PAGE], np.array(js) % PAGE
            for h in range(H):
                kk = decode(codes[pg, h, 0, of], fmt) * scales[pg, h, 0, None].astype(np.float64)
                vv = decode(codes[pg, h, 1, of], fmt) * scales[pg, h, 1, None].astype(np.float64)
                x = (kk @ q[row, h * G:(h + 1) * G].astype(np.float64).T) * scale
                p = np.exp(x - x.max(0))
                out[row, h * G:(h + 1) * G] = (p.T @ vv) / p.sum(0)[:, None]
                mag[row, h * G:(h + 1) * G] = (p.T @ np.abs(vv)) / p.sum(0)[:, None]
    return out, mag


def plan(lens, add, table, free, n_free, n_rows):
    """(table, lens_out, first, slots, pos, seq, status), one sequence after another."""
    table = table.copy()
    n, ld = table.shape
    first, lens_out = [0], []
    slots, pos, seq = (np.full(n_rows, -1, np.int64) for _ in range(3))
    asked = used = refused = row = 0
    for i in range(n):
        l, d = int(lens[i]), int(add[i])
        sane = l >= 0 and d >= 0
        rows = d if sane else 0
        ok = sane and l + d <= ld * PAGE and row + rows <= n_rows
        need = (l + d + PAGE - 1) // PAGE - (l + PAGE - 1) // PAGE if ok else 0
        before = asked
        asked += need
        if ok and need and asked > n_free:
            ok = False
        if ok:
            used += need
            for p in range(need):
                table[i, (l + PAGE - 1) // PAGE + p] = free[n_free - 1 - before - p]
        refused += not ok
        lens_out.append(l + d if ok else -1)
        for t in range(rows):
            if row + t >= n_rows:
                break
            seq[row + t] = i
            if ok:
                pos[row + t] = l + t
                page = int(table[i, (l + t) // PAGE])
                slots[row + t] = page * PAGE + (l + t) % PAGE if page >= 0 else -1
        row += rows
        first.append(row)
    return table, np.array(lens_out), np.minimum(first, 2**31 - 1), slots, pos, seq, np.array([n_free - used, refused])


def draw(x, t, k, p, m, u, mask=None):
    """(token, log probability) of one row."""
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -np.inf
    if mask is not None:
        x[mask == 0] = -np.inf
    x = np.minimum(x, float(np.finfo(np.float32).max))
    ids = np.nonzero(x > -np.inf)[0]
    if ids.size == 0:
        return -1, -np.inf
    order = ids[np.argsort(-x[ids], kind="stable")]
    if not t > 0:
        return int(order[0]), 0.0
    if k > 0:
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / t)
    below = np.cumsum(w) - w
    keep = np.ones(w.size, bool) if not p < 1 else below < p * w.sum()
    keep &= w >= m
    keep[0] = True
    kept = np.sort(order[keep])
    w = np.exp((x[kept] - x[order[0]]) / t)
    c = np.cumsum(w)
    u = min(max(float(np.float32(u)), 0.0), 1 - 2.0**-24) if u == u else 0.0
    at = min(int((c <= u * c[-1]).sum()), kept.size - 1)
    return int(kept[at]), float((x[kept[at]] - x[order[0]]) / t - np.log(c[-1]))
