"""64-bit statements of the paged latent cache's operators, for the tests, and how far a kernel may be from them.

`attention` returns besides the result the sum of absolute contributions of each output, of which the tolerances are
fractions: a kernel that forms scores and sums in 32 bits and rounds the weights and the result to the 16-bit type t is off by
at most
    eps/2 |out|                  the result's own rounding
  + eps/2 A                      the weights' rounding, A = sum_j p_j |v_j|
  + 2 e A                        an error e of the scores: a weight changes by e, and so does the sum it is divided by
  + 2^-18 A                      512 columns' products summed in 32 bits, exponentials (2^-22) and the division
with e = 576 * 2^-24 * scale * max_j sum_i |q_i c_ji|, the bound of a sum of 576 products in 32 bits; and lse by
e + 2^-20 (1 + |lse|).
"""
import math

import torch


def attention(q, cache, table, q_start, kv_len, scale, causal=True, window=0):
    """(out, lse, tol_out, tol_lse) in 64 bits; one sequence after the other. Tokens of no sequence: zeros and -inf."""
    T, H, D = q.shape
    ps = cache.shape[1]
    out = torch.zeros(T, H, 512, dtype=torch.float64, device=q.device)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    eps = torch.finfo(q.dtype).eps
    for b, kv in enumerate(kv_len.tolist()):
        t0, t1 = q_start[b].item(), q_start[b + 1].item()
        kv = min(max(kv, 0), table.shape[1] * ps)
        if t1 == t0 or kv == 0:
            continue
        pages = table[b, :-(-kv // ps)].long()
        ok = (pages >= 0) & (pages < cache.shape[0])
        rows = cache[pages.clamp(0, cache.shape[0] - 1)].double()
        rows[~ok] = 0
        rows = rows.reshape(-1, D)[:kv]
        x = q[t0:t1].double()
        s = torch.einsum("nhd,kd->nhk", x, rows) * scale
        size = torch.einsum("nhd,kd->nhk", x.abs(), rows.abs()) * scale
        p = kv - (t1 - t0) + torch.arange(t1 - t0, device=q.device)[:, None]
        j = torch.arange(kv, device=q.device)[None]
        seen = (j <= p) if causal else torch.ones(t1 - t0, kv, dtype=torch.bool, device=q.device)
        if window:
            seen = seen & (j > p - window)
        s = s.masked_fill(~seen[:, None], -math.inf)
        e = size.masked_fill(~seen[:, None], 0).amax(-1) * (576 * 2.0 ** -24)
        some = seen.any(-1)[:, None].expand(-1, H)
        lse[t0:t1] = torch.logsumexp(s, -1)
        w = torch.where(some[..., None], torch.softmax(s, -1), torch.zeros_like(s))
        out[t0:t1] = torch.einsum("nhk,kd->nhd", w, rows[:, :512])
        a = torch.einsum("nhk,kd->nhd", w, rows[:, :512].abs())
        tol[t0:t1] = eps / 2 * out[t0:t1].abs() + (eps / 2 + 2 * e[..., None] + 2.0 ** -18) * a
        tol_lse[t0:t1] = torch.where(some, e + 2.0 ** -20 * (1 + lse[t0:t1].abs()), torch.zeros_like(e))
    return out, lse, tol, tol_lse


def rotate(x, positions, freq, interleaved=False, mscale=1.0, inverse=False):
    """(out, tol): x [T, H, R]. 32-bit angles of less than half a turn, sine and cosine to two units in the last place and
    two products: 8 * 2^-24 of |x0| + |x1|, times mscale; then the rounding to x's type."""
    f = x.double()
    half = f.shape[-1] // 2
    a = positions.double()[:, None, None] * freq.double() * (-1 if inverse else 1)
    x0, x1 = (f[..., 0::2], f[..., 1::2]) if interleaved else (f[..., :half], f[..., half:])
    y0, y1 = mscale * (x0 * a.cos() - x1 * a.sin()), mscale * (x1 * a.cos() + x0 * a.sin())
    size = mscale * (x0.abs() + x1.abs()) * 8 * 2.0 ** -24
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat((u, v), -1))
    out = join(y0, y1)
    # the smallest step of a type with few exponent bits is absolute
    return out, torch.finfo(x.dtype).eps / 2 * out.abs() + join(size, size) + torch.finfo(x.dtype).smallest_normal \
        * torch.finfo(x.dtype).eps


class Pool:
    """The page rules in Python lists: lowest free page first, everything or nothing."""

    def __init__(self, table, length, refcount, page_size):
        self.table, self.length, self.count = table.tolist(), length.tolist(), refcount.tolist()
        self.ps, self.copies = page_size, []

    def _free(self):
        return [p for p, n in enumerate(self.count) if n == 0]

    def extend(self, seqs, new):
        need = [max(0, -(-n // self.ps) - -(-self.length[s] // self.ps)) for s, n in zip(seqs, new)]
        free = self._free()
        assert sum(need) <= len(free)
        for s, n, k in zip(seqs, new, need):
            have = -(-self.length[s] // self.ps)
            for i in range(k):
                page = free.pop(0)
                self.table[s][have + i] = page
                self.count[page] = 1
            self.length[s] = max(self.length[s], n)

    def fork(self, src, dst):
        free = [p for p in self._free()]
        for a, b in zip(src, dst):
            n = self.length[a]
            for i in range(n // self.ps):
                self.table[b][i] = self.table[a][i]
                self.count[self.table[a][i]] += 1
            if n % self.ps:
                page = free.pop(0)
                self.table[b][n // self.ps] = page
                self.count[page] = 1
                self.copies.append((self.table[a][n // self.ps], page))
            self.length[b] = n

    def free(self, seqs):
        for s in seqs:
            for i in range(-(-self.length[s] // self.ps)):
                self.count[self.table[s][i]] -= 1
                self.table[s][i] = -1
            self.length[s] = 0

    def compact(self):
        used = sum(n > 0 for n in self.count)
        holes = [p for p in range(used) if self.count[p] == 0]
        high = [p for p in range(used, len(self.count)) if self.count[p] > 0]
        to = dict(zip(high, holes))
        for s, n in enumerate(self.length):
            for i in range(-(-n // self.ps)):
                self.table[s][i] = to.get(self.table[s][i], self.table[s][i])
        for a, b in to.items():
            self.count[b], self.count[a] = self.count[a], 0
        self.copies += list(to.items())
