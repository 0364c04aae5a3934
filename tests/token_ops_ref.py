"""Plain statements of the operators on token ids, in 64 bits, one element after the other where order matters.  numpy only;
written from include/l3hip.h, sharing nothing with the kernels."""
import numpy as np

POOL, ROW, BAD, PAGE = 1, 2, 4, 8


def embed(ids, table, scale):
    """float64 (n, dim): scale * table[id], zeros for an id that is no row."""
    table = np.asarray(table, dtype=np.float64)
    out = np.zeros((len(ids), table.shape[1]))
    for t, i in enumerate(ids):
        if 0 <= i < table.shape[0]:
            out[t] = table[i] * scale
    return out


def embed_grad(ids, grad, rows, scale, old=None):
    """(sum, sum of absolute values, number of terms per row), float64; old: what the sum is added to."""
    grad = np.asarray(grad, dtype=np.float64)
    total = np.zeros((rows, grad.shape[1])) if old is None else np.array(old, dtype=np.float64)
    size = np.abs(total)
    count = np.zeros(rows, dtype=np.int64)
    for t, i in enumerate(ids):
        if 0 <= i < rows:
            total[i] += scale * grad[t]
            size[i] += np.abs(scale * grad[t])
            count[i] += 1
    return total, size, count


class Cache:
    """The state of a paged cache: python lists."""

    def __init__(self, length, held, table, free, n_free, page, n_pages, max_pages):
        self.length, self.held = list(length), list(held)
        self.table = [list(r) for r in table]
        self.free = list(free)
        self.n_free = n_free
        self.page, self.n_pages, self.max_pages = page, n_pages, max_pages

    def _sane(self, i):
        return 0 <= self.held[i] <= self.max_pages and 0 <= self.length[i] <= self.held[i] * self.page

    def slots(self, off, cap, slots, pos):
        """Fills slots / pos (lists of cap entries) and returns the status."""
        status = 0
        pool = self.n_free
        if not 0 <= pool <= self.n_pages:
            status, pool = BAD, 0
        asked = 0
        left = pool
        for i in range(len(self.length)):
            a, b = off[i], off[i + 1]
            ok = True
            need = 0
            if a > b or b > cap or not self._sane(i):
                status, ok = status | BAD, False
            elif b > a:
                end = self.length[i] + b - a
                if end > self.max_pages * self.page or end >= 2 ** 31:
                    status, ok = status | ROW, False
                else:
                    need = max(0, -(-end // self.page) - self.held[i])
                    asked += need
                    if need and asked > pool:
                        status, ok = status | POOL, False
            if ok:
                for j in range(need):
                    left -= 1
                    self.table[i][self.held[i] + j] = self.free[left]
                self.held[i] += need
            for t in range(a, min(b, cap)):
                p = self.length[i] + t - a
                slots[t] = pos[t] = -1
                if ok:
                    pos[t] = p
                    page = self.table[i][p // self.page]
                    if 0 <= page < self.n_pages:
                        slots[t] = page * self.page + p % self.page
                    else:
                        status |= PAGE
            if ok:
                self.length[i] += b - a
        if 0 <= self.n_free <= self.n_pages:
            self.n_free = left
        return status

    def trim(self, keep):
        status = 0
        usable = 0 <= self.n_free <= self.n_pages
        if not usable:
            status = BAD
        room = self.n_pages - self.n_free if usable else 0
        start = self.n_free
        asked = 0
        for i in range(len(self.length)):
            if keep[i] < 0:
                continue
            if not self._sane(i):
                status |= BAD
                continue
            now = min(keep[i], self.length[i])
            stay = -(-now // self.page)
            give = self.held[i] - stay
            asked += give
            if give and asked > room:
                status |= POOL
                continue
            for j in range(stay, self.held[i]):
                self.free[self.n_free] = self.table[i][j]
                self.n_free += 1
            self.length[i], self.held[i] = now, stay
        assert start == self.n_free or usable
        return status


def verify(draft, off, max_draft, target, q, vocab, u_accept, u_draw):
    """(out (n, max_draft + 1), accepted (n)); target, q: float64 rows."""
    n = len(off) - 1
    out = np.full((n, max_draft + 1), -1, dtype=np.int64)
    accepted = np.full(n, -1, dtype=np.int64)

    def clean(w):
        with np.errstate(invalid="ignore"):
            return np.where((w > 0) & np.isfinite(w), w, 0.0)

    for i in range(n):
        lo, hi = int(off[i]), int(off[i + 1])
        if lo > hi or hi > len(draft) or hi - lo > max_draft:
            continue
        a = 0
        while a < hi - lo:
            d = int(draft[lo + a])
            if not 0 <= d < vocab:
                break
            qd = 1.0 if q is None else q[lo + a][d]
            if not float(u_accept[lo + a]) * qd < target[lo + i + a][d]:
                break
            out[i, a] = d
            a += 1
        accepted[i] = a
        p = target[lo + i + a]
        w = full = clean(p)
        if a < hi - lo:
            if q is None:
                w = full.copy()
                if 0 <= draft[lo + a] < vocab:
                    w[draft[lo + a]] = 0.0
            else:
                with np.errstate(invalid="ignore"):
                    w = clean(p - q[lo + a])
            if w.sum() == 0:
                w = full
        c = np.cumsum(w)
        if c[-1] > 0:
            at = np.nonzero(c > float(u_draw[i]) * c[-1])[0]
            out[i, a] = at[0] if len(at) else np.nonzero(w)[0][-1]
    return out, accepted
