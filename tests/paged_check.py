"""Plain models for the paged cache's tests: the pool's bookkeeping with Python
lists, and the windowed attention's definition in 64 bits with the bounds that its
kernel's roundings allow."""
import math

import torch

DIM, NOPE = 512, 448


def quantized_rows(n, seed, device, outliers=0.01):
    """Cache arrays of n rows ~N(0,1), a share of them eight times as large."""
    g = torch.Generator(device).manual_seed(seed)
    x = torch.randn((n, DIM), generator=g, device=device)
    x *= torch.where(torch.rand((n, 1), generator=g, device=device) < outliers, 8.0, 1.0)
    b = x[:, :NOPE].reshape(n, 7, 64)
    e = torch.ceil(torch.log2(b.abs().amax(-1).clamp_min(1e-4) / 448.0))
    codes = (b * torch.exp2(-e)[..., None]).reshape(n, NOPE).to(torch.float8_e4m3fn).view(torch.uint8)
    sexp = torch.zeros((n, 8), dtype=torch.int8, device=device)
    sexp[:, :7] = e.to(torch.int8)
    return codes.contiguous(), sexp, x[:, NOPE:].half().contiguous()


def row_values(codes, sexp, tail):
    """Rows in 64 bits, from the bits of the format (code 0x7F / 0xFF: NaN)."""
    c = codes.to(torch.int64)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m / 512.0, (1.0 + m / 8.0) * torch.exp2((e - 7).double()))
    v = torch.where((c & 127) == 127, math.nan, v)
    v = torch.where(c >= 128, -v, v) * torch.exp2(sexp[..., :7].double()).repeat_interleave(64, -1)
    return torch.cat([v.half().double(), tail.view(torch.float16).double()], -1)


def attend_64(q, kv, positions, window, first, sinks):
    """q [n, heads, 512] at `positions` over one sequence's rows kv, in 64 bits: the
    outputs, the same averages of |value|, how far each head's scores may be off, and the
    largest weight times the sum of |value|."""
    n = q.shape[0]
    k = torch.arange(kv.shape[0], device=q.device)[None]
    p = torch.as_tensor(positions, device=q.device)[:, None]
    seen = k <= p
    if window:
        seen &= (k > p - window) | (k < first)
    out, size, all_of, err = *(torch.zeros_like(q, dtype=torch.float64) for _ in range(3)), []
    for i in range(n):
        rows = kv[seen[i]]
        if rows.shape[0] == 0:
            err.append(torch.zeros(q.shape[1], dtype=torch.float64, device=q.device))
            continue
        x = q[i].double()
        s = x @ rows.T / math.sqrt(DIM)
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None]], -1)
        w = torch.softmax(s, -1)[:, :rows.shape[0]]
        out[i] = w @ rows
        size[i] = w @ rows.abs()
        all_of[i] = w.amax(-1, keepdim=True) * rows.abs().sum(0)
        # |error of a score| <= 42 steps of 2^-23 (16 matrix instructions a score, each sum
        # of 32 products in 5 levels, truncated at worst) of the sum of |q k|
        err.append(42 * 2.0 ** -23 * (x.abs() @ rows.abs().T / math.sqrt(DIM)).amax(-1) + 2.0 ** -22 * s.abs().amax(-1))
    return out, (size, all_of), torch.stack(err) if err else torch.zeros((0, q.shape[1]), dtype=torch.float64, device=q.device)


def bound_of(ref, size, err, f32):
    """A weight is off by its own rounding (one f16: 2^-11; hi + lo: 2^-22) and by its
    score's error, as a share of itself; numerator and denominator each, so twice the
    average |value|. One that is subnormal in f16 is off by up to 2^-25 instead, where the largest weight is
    2^-8 or more (hi + lo: 2^8): by 2^-17 (2^-33) of the largest, for each row. Then the
    result's own rounding (bf16 2^-8, fp32 2^-24)."""
    size, all_of = size
    weight = (2.0 ** -22 if f32 else 2.0 ** -11) + err[..., None]
    return 2 * weight * size + 2 * (2.0 ** -33 if f32 else 2.0 ** -17) * all_of + \
        (2.0 ** -24 if f32 else 2.0 ** -8) * ref.abs() + 1e-30


class PoolModel:
    """The pool as lists; contents[layer][row] is a tag."""

    def __init__(self, n_pages, page_rows, n_seqs, entries, layers):
        self.page, self.entries = page_rows, entries
        self.refs, self.rows = [0] * n_pages, [0] * n_seqs
        self.table = [[] for _ in range(n_seqs)]
        self.tags = [[0] * (n_pages * page_rows) for _ in range(layers)]

    def n(self, rows):
        return -(-rows // self.page)

    def _take(self, want):
        free = [p for p, r in enumerate(self.refs) if r == 0]
        return free[:want] if len(free) >= want else None

    def extend(self, seqs, n_new, n_dst):
        none = [-1] * n_dst
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.rows) for s in seqs) or min(n_new, default=0) < 0:
            return -22, none
        if any(k and self.rows[s] % self.page and self.refs[self.table[s][-1]] != 1 for s, k in zip(seqs, n_new)):
            return -22, none
        if sum(n_new) > n_dst:
            return -22, none
        if any(self.n(self.rows[s] + k) > self.entries for s, k in zip(seqs, n_new)):
            return -28, none
        need = [self.n(self.rows[s] + k) - self.n(self.rows[s]) for s, k in zip(seqs, n_new)]
        pages = self._take(sum(need))
        if pages is None:
            return -28, none
        dst = []
        for s, k, m in zip(seqs, n_new, need):
            mine, pages = pages[:m], pages[m:]
            for p in mine:
                self.refs[p] = 1
            self.table[s] += mine
            for r in range(self.rows[s], self.rows[s] + k):
                dst.append(self.table[s][r // self.page] * self.page + r % self.page)
            self.rows[s] += k
        return 0, dst + [-1] * (n_dst - len(dst))

    def fork(self, parents, children, n_rows, deep):
        rows = list(self.rows)
        take = []
        if len(set(children)) < len(children):
            return -22
        for i, (a, b) in enumerate(zip(parents, children)):
            if not (0 <= a < len(rows) and 0 <= b < len(rows)) or rows[b]:
                return -22
            r = rows[a] if n_rows is None or n_rows[i] < 0 else n_rows[i]
            if r > rows[a]:
                return -22
            take.append((a, b, r, self.n(r) if deep else int(r % self.page != 0)))
        pages = self._take(sum(t[3] for t in take))
        if pages is None:
            return -28
        tables = [list(t) for t in self.table]
        for a, b, r, k in take:
            mine, pages = pages[:k], pages[k:]
            held = tables[a][:self.n(r)]
            for p in held[:len(held) - k]:
                self.refs[p] += 1
            for i, (old, new) in enumerate(zip(held[len(held) - k:], mine)):
                self.refs[new] = 1
                used = min(self.page, r - (len(held) - k + i) * self.page)
                for tags in self.tags:
                    tags[new * self.page:new * self.page + used] = tags[old * self.page:old * self.page + used]
            self.table[b] = held[:len(held) - k] + mine
            self.rows[b] = r
        return 0

    def free(self, seqs, keep):
        keep = [0] * len(seqs) if keep is None else keep
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.rows) for s in seqs):
            return -22
        for s, k in zip(seqs, keep):
            if not 0 <= k <= self.rows[s]:
                return -22
            if k < self.rows[s] and k % self.page and self.refs[self.table[s][k // self.page]] != 1:
                return -22
        for s, k in zip(seqs, keep):
            for p in self.table[s][self.n(k):]:
                self.refs[p] -= 1
            self.table[s], self.rows[s] = self.table[s][:self.n(k)], k
        return 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        src = [p for p, r in enumerate(self.refs) if r > 0 and p >= live]
        dst = [p for p, r in enumerate(self.refs) if r == 0 and p < live]
        now = dict(zip(src, dst))
        for a, b in now.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for tags in self.tags:
                tags[b * self.page:(b + 1) * self.page] = tags[a * self.page:(a + 1) * self.page]
        self.table = [[now.get(p, p) for p in t] for t in self.table]
        return live
