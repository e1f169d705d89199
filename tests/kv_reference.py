"""The paged key/value cache restated in plain torch, 64 bits and Python lists: what tests/test_gpu_kvcache.py holds the kernels to."""
import torch


def norm_rotate(x, weight, cos, sin, pos, eps):
    """x [T, H, D] -> float64: x / rms(x) * weight per head, then the first 2 * cos.shape[1] dimensions turned by cos / sin[pos]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    if cos is None:
        return x
    h = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h:]], -1)


def attention(q, k, v, pos, window, sinks, scale, there=None):
    """q [n, H, D] at positions pos [n], keys k, v [L, G, D] at positions 0 .. L - 1 (`there` [L]: which exist) -> (out [n, H, D], the
    mean of |v| under the same weights, the largest sum over d of |q_d k_d| of a visible pair): float64.  Only what a query sees enters.
    The middle one carries, as .rounded_keys, how far out moves (first order) when each product q_d k_d is off by a share of itself: the
    weighted mean of |v - out| sum |q_d k_d| scale, per unit of that share."""
    n, H, D = q.shape
    L, G, _ = k.shape
    out = torch.zeros((n, H, D), dtype=torch.float64, device=q.device)
    mag, moved, dot = torch.zeros_like(out), torch.zeros_like(out), 0.0
    at = torch.arange(L, device=q.device)
    for i in range(n):
        see = at <= pos[i]
        if window > 0:
            see &= (at > pos[i] - window) | (at < sinks)
        if there is not None:
            see &= there
        idx = see.nonzero().view(-1)
        if not len(idx):
            continue
        kk, vv = k[idx].double(), v[idx].double()
        for h in range(H):
            g = h // (H // G)
            prod = kk[:, g] * q[i, h].double()
            x = prod.sum(-1) * scale
            w = torch.softmax(x, 0)
            out[i, h] = w @ vv[:, g]
            mag[i, h] = w @ vv[:, g].abs()
            dots = prod.abs().sum(-1)
            moved[i, h] = (w * dots * scale) @ (vv[:, g] - out[i, h]).abs()
            dot = max(dot, float(dots.max()))
    mag.rounded_keys = moved
    return out, mag, dot


class Pages:
    """Table, lengths and counts by the rules of include/q3c.h, on Python lists."""

    def __init__(self, pages, page_size, rows, width):
        self.P, self.ps, self.W = pages, page_size, width
        self.table = [[-1] * width for _ in range(rows)]
        self.lens, self.refs = [0] * rows, [0] * pages
        self.status = 0

    def _take(self):
        for p, r in enumerate(self.refs):
            if r == 0:
                self.refs[p] = 1
                return p
        self.status |= 2
        return -1

    def reserve(self, rows, counts):
        seen = set()
        for r, n in zip(rows, counts):
            if not 0 <= r < len(self.lens) or r in seen:
                self.status |= 1
                continue
            seen.add(r)
            old, cap = self.lens[r], self.W * self.ps
            self.lens[r] = old + n
            if old + n > cap:
                self.status |= 8
            for j in range(-(-min(old, cap) // self.ps), -(-min(old + n, cap) // self.ps)):
                self.table[r][j] = self._take()

    def _drop(self, r, j):
        p = self.table[r][j]
        self.table[r][j] = -1
        if p >= 0:
            self.refs[p] -= 1

    def release(self, rows):
        for r in rows:
            if not 0 <= r < len(self.lens):
                self.status |= 1
                continue
            for j in range(self.W):
                self._drop(r, j)
            self.lens[r] = 0

    def trim(self, rows, window, sinks):
        for r in rows:
            for j in range(self.W):
                if j * self.ps >= sinks and (j + 1) * self.ps <= self.lens[r] - window:
                    self._drop(r, j)

    def fork(self, parents, children):
        """-> pages that are copied, [(source, destination)]"""
        good = []
        for i, (u, c) in enumerate(zip(parents, children)):
            ok = 0 <= u < len(self.lens) and 0 <= c < len(self.lens) and c not in children[:i] and u not in children and self.lens[c] == 0
            self.status |= 0 if ok else 1
            good.append(ok)
        pairs, grants = [], []
        for u, c, ok in zip(parents, children, good):
            n = min(self.lens[u], self.W * self.ps) if ok else 0
            src = self.table[u][n // self.ps] if n % self.ps else -1
            dst = self._take() if src >= 0 else -1
            grants.append(dst)
            if dst >= 0:
                pairs.append((src, dst))
        for u, c, ok, dst in zip(parents, children, good, grants):
            if not ok:
                continue
            n = min(self.lens[u], self.W * self.ps)
            full = n // self.ps
            for j in range(self.W):
                p = self.table[u][j] if j < full else dst if j == full else -1
                if j < full and p >= 0:
                    self.refs[p] += 1
                self.table[c][j] = p
            self.lens[c] = n
        return pairs

    def copy(self, src, dst):
        pairs = []
        for i, (s, d) in enumerate(zip(src, dst)):
            if not (0 <= s < self.P and 0 <= d < self.P) or (s != d and s in dst):
                self.status |= 4
            elif d not in dst[i + 1:] and s != d:
                pairs.append((s, d))
        return pairs

    def compact(self):
        live = [p for p in range(self.P) if self.refs[p] > 0]
        n = len(live)
        src, dst = [p for p in live if p >= n], [p for p in range(n) if self.refs[p] <= 0]
        to = dict(zip(src, dst))
        for t in self.table:
            t[:] = [to.get(p, p) for p in t]
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
        return list(to.items()), n
