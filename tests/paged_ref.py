"""Plain restatements of the serving operators in numpy: tables from lengths,
appended codes, attention and sampling in 64 bits."""
import numpy as np


class Tables:
    """What PageTable does, one request after another."""

    def __init__(self, requests, max_pages, num_pages, page):
        self.page, self.max_pages = page, max_pages
        self.pages = np.full((requests, max_pages), -1, np.int64)
        self.held = np.zeros(requests, np.int64)
        self.free = list(range(num_pages - 1, -1, -1))

    def plan(self, lens, new, rows):
        n = len(lens)
        start, after = [0], []
        req, pos, slots = (np.full(rows, -1, np.int64) for _ in range(3))
        at, asked, height = 0, 0, len(self.free)
        for r in range(n):
            base, m = max(int(lens[r]), 0), max(int(new[r]), 0)
            ok = base + m <= self.max_pages * self.page and at + m <= rows
            want = max(0, -(-(base + m) // self.page) - self.held[r]) if ok else 0
            asked += want
            ok = ok and (want == 0 or asked <= height)
            if ok:
                for _ in range(want):
                    self.pages[r, self.held[r]] = self.free.pop()
                    self.held[r] += 1
            for j in range(m):
                if at + j < rows:
                    req[at + j] = r
                    if ok:
                        p = base + j
                        pos[at + j] = p
                        slots[at + j] = self.pages[r, p // self.page] * self.page + p % self.page
            at += m
            start.append(min(at, rows))
            after.append(base + m if ok else base)
        return dict(row_start=np.array(start), lens=np.array(after), request=req, positions=pos, slots=slots)

    def release(self, done):
        for r in np.nonzero(done)[0]:
            self.free += list(self.pages[r, :self.held[r]])
            self.pages[r] = -1
            self.held[r] = 0


def half_away(x):
    return np.sign(x) * np.floor(np.abs(x) + 0.5)


def append(codes, scales, x, slots):
    """codes [pages, heads, page, hd] (float64 integers) and fp32 scales, in
    place; x [rows, heads, hd] float64 holding fp32 values."""
    page = codes.shape[2]
    i = 0
    while i < len(slots):
        if slots[i] < 0 or slots[i] >= codes.shape[0] * page:
            i += 1
            continue
        j = i + 1
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % page:
            j += 1
        pg, off = slots[i] // page, slots[i] % page
        for h in range(codes.shape[1]):
            v = x[i:j, h]
            fin = np.abs(v[np.isfinite(v)])
            big = fin.max() if fin.size else 0.0
            own = np.float32(0) if big < 2.0 ** -100 else np.float32(np.float32(big) / np.float32(127))
            old = scales[pg, h] if off else np.float32(0)
            new = max(old, own)
            if off and new > old:
                codes[pg, h, :off] = half_away(codes[pg, h, :off] * float(old) / float(new))
            with np.errstate(invalid="ignore", divide="ignore"):
                c = half_away(v / float(new)) if new > 0 else np.zeros_like(v)
            codes[pg, h, off:off + j - i] = np.where(np.isnan(v), 0, np.clip(np.nan_to_num(c, posinf=127, neginf=-127), -127, 127))
            scales[pg, h] = new
        i = j


def attention(q, kc, vc, ks, vs, pages, start, positions, scale):
    """float64 attention; kc [pages, heads, page, hd], vc [pages, heads, hd, page].
    Rows of no request are NaN."""
    rows, heads, hd = q.shape
    kv, page = kc.shape[1:3]
    out = np.full((rows, heads, hd), np.nan)
    for r in range(len(start) - 1):
        for t in range(start[r], start[r + 1]):
            n = min(positions[t] + 1, pages.shape[1] * page)
            ids = pages[r, np.arange(max(n, 0)) // page]
            ok = (ids >= 0) & (ids < kc.shape[0])
            ids, off = ids[ok], (np.arange(max(n, 0)) % page)[ok]
            for h in range(heads):
                g = h // (heads // kv)
                k = kc[ids, g, off].astype(np.float64) * ks[ids, g].astype(np.float64)[:, None]
                v = vc[ids, g, :, off].astype(np.float64) * vs[ids, g].astype(np.float64)[:, None]
                if not len(ids):
                    out[t, h] = 0
                    continue
                s = k @ q[t, h] * scale
                p = np.exp(s - s.max())
                out[t, h] = p @ v / p.sum()
    return out


def sample(x, t, k, p, mp, u):
    """One row's token."""
    if not t > 0:
        return 0 if np.isnan(x[0]) else int(np.where(np.isnan(x), -np.inf, x).argmax())
    x = np.minimum(np.where(np.isnan(x), -np.inf, x.astype(np.float64)), np.finfo(np.float32).max)
    if x.max() == -np.inf:
        return 0
    w = np.exp((x - x.max()) / float(t))
    w[w < np.exp(-32.0)] = 0.0
    rank = np.lexsort((np.arange(len(x)), -x))
    n = min(int(k), len(x)) if k > 0 else len(x)
    mass = np.cumsum(w[rank[:n]])
    if p < 1:
        n = min(n, int(np.searchsorted(mass, max(float(p), 0.0) * mass[-1])) + 1)
    if mp > 0:
        n = max(1, min(n, int((w >= min(float(mp), 1.0)).sum())))
    kept = np.sort(rank[:n])
    mass = np.cumsum(w[kept])
    i = int(np.searchsorted(mass, float(u) * mass[-1], side="right"))
    return int(kept[min(i, int(np.nonzero(w[kept])[0][-1]))])
