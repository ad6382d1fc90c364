"""The 8-bit cache in 64 bits on the CPU, from its definitions: the checker of
test_gpu_fp8.py."""
from __future__ import annotations

import math

import torch


def scale_for(amax: float) -> float:
    """2^e, e >= -126 the smallest with amax <= 448 * 2^e."""
    e = -126
    if amax > 0:
        e = max(-126, math.frexp(amax)[1] - 12)
        while amax > 448.0 * 2.0 ** e:
            e += 1
    return 2.0 ** e


def round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value, ties to even, +-448 beyond; NaN stays NaN."""
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(2.0 ** -6, 512.0))) - 3)
    r = torch.round(a / step) * step
    return torch.where(torch.isnan(y), y, torch.sign(y) * r.clamp_max(448.0))


class RefPool:
    """codes [2, NB, H, bs, D] and scales [2, NB, H] as float64, mass [NB, H, bs]."""

    def __init__(self, codes, scales, mass=None):
        self.codes, self.scales = codes.float().cpu().double(), scales.cpu().double()
        self.mass = None if mass is None else mass.cpu().double()
        self.bs = codes.shape[3]

    def append(self, k, v, slots) -> None:
        rows: dict[int, dict[int, int]] = {}
        for i, s in enumerate(slots.tolist()):
            if 0 <= s < self.codes.shape[1] * self.bs:
                rows.setdefault(s // self.bs, {})[s % self.bs] = i  # the later token counts
        for blk, at in rows.items():
            for p, x in enumerate((k, v)):
                x = x.cpu().double()
                for h in range(x.shape[1]):
                    new = torch.stack([x[i, h] for i in at.values()])
                    fin = new[torch.isfinite(new)].abs()
                    old = 0.0 if 0 in at else float(self.scales[p, blk, h])
                    s = max(old, scale_for(float(fin.max()) if fin.numel() else 0.0))
                    if 0 not in at and s > old > 0:
                        self.codes[p, blk, h] = round_e4m3(self.codes[p, blk, h] * (old / s))
                    for r, i in at.items():
                        self.codes[p, blk, h, r] = round_e4m3(x[i, h] / s)
                    self.scales[p, blk, h] = s
            if self.mass is not None:
                for r in at:
                    self.mass[blk, :, r] = 0.0

    def rows(self, p, table, pos):
        blk = table.long()[pos // self.bs]
        return self.codes[p][blk, :, pos % self.bs] * self.scales[p][blk][..., None]  # [n, H, D]

    def decode(self, q, tables, lens, scale, softcap=0.0, slopes=None, window=0, accumulate=False):
        """(out, bound): bound is how far a float32 computation may be off.

        A score is a float32 sum of D products, rounded or truncated at most
        D / 16 + 8 times: off by at most g * S, g = (D / 16 + 8) 2^-23, S the
        largest sum of magnitudes (scale * sum |q k|, plus the bias).  That is
        the weight's relative error, met once in the numerator and once in the
        denominator; exp2, the split of a weight into two halves and the
        sums over L tokens add (L / 32 + 24) 2^-23.  A weight is held as two
        f16 numbers in units in which the row's largest is 2^14 or more and
        the block's scale is relative to the largest scale s_max: whatever is
        below f16's smallest step, 2^-24, is rounded, which is at most 2^-25,
        so a token adds at most 2^-39 s_max |code| (of the row's largest
        weight, which is at most 1) to an output that it may be light in."""
        q = q.cpu().double()
        B, hq, D = q.shape
        H = self.codes.shape[2]
        out, bound = torch.zeros(B, hq, D, dtype=torch.float64), torch.zeros(B, hq, D, dtype=torch.float64)
        self.mass_bound = None if self.mass is None else self.mass.abs() * 2.0 ** -22
        for b in range(B):
            L = int(lens[b])
            if L == 0:
                continue
            pos = torch.arange(max(0, L - window) if window else 0, L)
            k, v = (self.rows(p, tables[b].cpu(), pos) for p in range(2))
            blk = tables[b].cpu().long()[pos // self.bs]
            s_max = self.scales[1][blk].amax(0)
            for h in range(H):
                g0, g1 = h * (hq // H), (h + 1) * (hq // H)
                z = scale * q[b, g0:g1] @ k[:, h].t()
                S = (abs(scale) * q[b, g0:g1].abs() @ k[:, h].abs().t()).amax(1)
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                if slopes is not None:
                    bias = slopes.cpu().double()[g0:g1, None] * (pos - (L - 1))
                    z = z + bias
                    S = S + bias.abs().amax(1)
                p = torch.softmax(z, 1)
                rel = 2 * (D / 16 + 8) * 2.0 ** -23 * S + (L / 32 + 24) * 2.0 ** -23
                out[b, g0:g1] = p @ v[:, h]
                bound[b, g0:g1] = rel[:, None] * (p @ v[:, h].abs()) + 1e-37 + \
                    2.0 ** -39 * s_max[h] * self.codes[1][blk, h, pos % self.bs].abs().sum(0)
                if accumulate:
                    self.mass[blk, h, pos % self.bs] += p.sum(0)
                    self.mass_bound[blk, h, pos % self.bs] += (rel[:, None] * p).sum(0) + 2.0 ** -23 * p.sum(0)
        return out, bound

    def evict(self, tables, lens, new_tables, budget, recent):
        B, H = tables.shape[0], self.codes.shape[2]
        kept = torch.full((B, H, budget), -1, dtype=torch.int32)
        new_lens = torch.zeros(B, dtype=torch.int32)
        before = (self.codes.clone(), self.scales.clone(), self.mass.clone())
        for b in range(B):
            L = int(lens[b])
            m = new_lens[b] = min(L, budget)
            old = max(0, L - recent)
            for h in range(H):
                pos = torch.arange(L)
                blk = tables[b].cpu().long()[pos // self.bs]
                w = before[2][blk, h, pos % self.bs]
                order = sorted(range(old), key=lambda t: (-math.inf if math.isnan(w[t]) else -float(w[t]), t))
                order = [t for t in order if math.isnan(w[t])] + [t for t in order if not math.isnan(w[t])]
                keep = sorted(order[: int(m) - (L - old)] + list(range(old, L)))
                kept[b, h, : int(m)] = torch.tensor(keep, dtype=torch.int32)
                for j in range(0, int(m), self.bs):
                    part = keep[j:j + self.bs]
                    dst = int(new_tables[b, j // self.bs])
                    src = [(int(tables[b, t // self.bs]), t % self.bs) for t in part]
                    for p in range(2):
                        s = max(float(before[1][p, k, h]) for k, _ in src)
                        for r, (k, o) in enumerate(src):
                            c = before[0][p, k, h, o]
                            f = float(before[1][p, k, h])
                            self.codes[p, dst, h, r] = c if f == s else round_e4m3(c * (f / s))
                        self.scales[p, dst, h] = s
                    for r, (k, o) in enumerate(src):
                        self.mass[dst, h, r] = before[2][k, h, o]
        return kept, new_lens
