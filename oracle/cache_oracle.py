"""The operators around a paged key/value cache from their definitions, in 64 bits on the CPU, one row or page at a time."""
import math

import torch


def rotary(x, phase, interleaved, magnitude=1.0):
    """x [..., D], phase [..., pairs] (broadcast): pairs of channels times exp(i phase)."""
    r = 2 * phase.shape[-1]
    x = x.double()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2: r])
    u, w = magnitude * (a * phase.cos() - b * phase.sin()), magnitude * (a * phase.sin() + b * phase.cos())
    y = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.cat([y, x[..., r:]], -1)


def rotary_size(x, pairs, interleaved):
    """|a| + |b| of each channel's pair, 0 for the channels behind them: what the 32-bit products' errors grow with."""
    r = 2 * pairs
    x = x.double().abs()
    if interleaved:
        s = (x[..., 0:r:2] + x[..., 1:r:2]).repeat_interleave(2, -1)
    else:
        s = (x[..., : r // 2] + x[..., r // 2: r]).repeat(*[1] * (x.dim() - 1), 2)
    return torch.cat([s, torch.zeros_like(x[..., r:])], -1)


def rows(lengths, cu):
    """(sequence, position) of every packed token; None where it belongs to no sequence."""
    out = {}
    for i, n in enumerate(lengths):
        for t in range(cu[i], cu[i + 1]):
            out[t] = (i, n - cu[i + 1] + t)
    return out


def attention(q, k_pages, v_pages, table, lengths, cu, causal, scale):
    """(out, lse, weight): weight [T, heads, D] is sum of softmax |v|, what the rounding of the probabilities grows with."""
    T, H, D = q.shape
    Hkv, ps = k_pages.shape[1], k_pages.shape[2]
    out, weight = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    size = torch.zeros(T, H, dtype=torch.float64)      # max over keys of sum |q k| scale
    for i, n in enumerate(lengths):
        a, b = cu[i], cu[i + 1]
        if a == b or n == 0:
            continue
        pages = table[i][: -(-n // ps)]
        k = k_pages[pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :n].double().repeat_interleave(H // Hkv, 0)
        v = v_pages[pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :n].double().repeat_interleave(H // Hkv, 0)
        x = q[a:b].double().transpose(0, 1) @ k.transpose(1, 2) * scale
        last = torch.arange(n - (b - a), n) if causal else torch.full((b - a,), n - 1)
        see = torch.arange(n) <= last[:, None]
        x = x.masked_fill(~see, -math.inf)
        z = torch.logsumexp(x, -1)
        p = torch.where(see, torch.exp(x - z[..., None]), torch.zeros((), dtype=torch.float64))
        out[a:b] = (p @ v).transpose(0, 1)
        weight[a:b] = (p @ v.abs()).transpose(0, 1)
        lse[a:b] = z.T
        size[a:b] = (q[a:b].double().abs().transpose(0, 1) @ k.abs().transpose(1, 2)).amax(-1).T * abs(scale)
    return out, lse, weight, size


class Pool:
    """Tables and counts as lists; pages as a tensor [slices, pages, ...] that the steps below change in place."""

    def __init__(self, table, lens, refs, pages, page_size):
        self.table, self.lens, self.refs = [list(r) for r in table], list(lens), list(refs)
        self.pages, self.ps = pages, page_size

    def used(self, n):
        return -(-n // self.ps)

    def allocate(self, new):
        free, need, served = self.refs.count(0), 0, []
        for i, x in enumerate(new):
            want = self.used(self.lens[i] + x) - self.used(self.lens[i]) if x >= 0 else 0
            if x < 0 or self.lens[i] + x > len(self.table[i]) * self.ps:
                served.append(False)
                continue
            need += want
            served.append(want == 0 or need <= free)
        for i, x in enumerate(new):
            if served[i]:
                for e in range(self.used(self.lens[i]), self.used(self.lens[i] + x)):
                    self.table[i][e] = self.refs.index(0)
                    self.refs[self.table[i][e]] = 1
                self.lens[i] += x
        return served

    def free(self, which):
        for s in which:
            if 0 <= s < len(self.table):
                for p in self.table[s]:
                    if p >= 0:
                        self.refs[p] -= 1
                self.table[s], self.lens[s] = [-1] * len(self.table[s]), 0

    def fork(self, src, dst):
        served, rows = [], {}
        free = [p for p, r in enumerate(self.refs) if r == 0]
        for i, (s, d) in enumerate(zip(src, dst)):
            there = lambda n: 0 <= n < len(self.table)  # noqa: E731
            # a later pair with the same destination has it, unless that one is skipped
            if not (there(s) and there(d)) or any(y == d and there(x) for x, y in zip(src[i + 1:], dst[i + 1:])):
                served.append(False)
                continue
            served.append(True)
            if s == d:
                continue
            u = self.used(self.lens[s])
            row = self.table[s][:u] + [-1] * (len(self.table[s]) - u)
            if self.lens[s] % self.ps:
                if not free:
                    served[-1] = False
                    continue
                row[u - 1] = free.pop(0)
                self.pages[:, row[u - 1]] = self.pages[:, self.table[s][u - 1]]
            rows[d] = (row, self.lens[s])
        for d, (row, n) in rows.items():
            for p in row:
                if p >= 0:
                    self.refs[p] += 1
        for d, (row, n) in rows.items():
            for p in self.table[d]:
                if p >= 0:
                    self.refs[p] -= 1
        for d, (row, n) in rows.items():
            self.table[d], self.lens[d] = row, n
        return served

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        to = {}
        for p in range(live, len(self.refs)):
            if self.refs[p] > 0:
                to[p] = holes.pop(0)
                self.pages[:, to[p]] = self.pages[:, p]
                self.refs[to[p]], self.refs[p] = self.refs[p], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return live
