"""Trees of drafted tokens for the tests of the operators that deal with them."""
import random

import torch

from tests.paged_util import Batch


def random_parents(news, spread, seed, roots=0.0):
    """Parents of the packed rows of sequences with `news` rows: one of the `spread` rows before, or none for row 0 and a few others."""
    r, out = random.Random(seed), []
    for n in news:
        out += [-1 if i == 0 or r.random() < roots else i - 1 - r.randrange(min(i, spread)) for i in range(n)]
    return out


def branch(parents, i):
    """Row i and its ancestors, `parents` those of its sequence; a parent that is no earlier row is none."""
    rows = []
    while i >= 0:
        rows.append(i)
        i = parents[i] if 0 <= parents[i] < i else -1
    return rows


class TreeBatch(Batch):
    """A `Batch` whose packed rows are trees: `attention` and so `check` are those of the branches."""

    def __init__(self, seqs, *args, parents=None, spread=4, roots=0.0, **kw):
        super().__init__(seqs, *args, **kw)
        self.parent_list = random_parents([n for n, _ in seqs], spread, kw.get("seed", 0), roots) if parents is None else list(parents)
        self.parents = torch.tensor(self.parent_list, dtype=torch.int32, device=self.device)

    def attention(self, scale=None):
        """As Batch.attention, row by row of what its branch has; a sequence at a time with a mask of its own."""
        out, lse, mass, size = super().attention(scale)
        scale = self.dim ** -0.5 if scale is None else scale
        group = self.hq // self.hkv
        for b, (n, length) in enumerate(self.seqs):
            if n == 0 or length <= 0:
                continue
            (k, there), (v, _) = self.stored(b, 0), self.stored(b, 1)
            lo = self.cu_list[b]
            see = torch.zeros(n, length, dtype=torch.bool)
            see[:, :max(length - n, 0)] = True
            for i in range(n):
                if length - n + i < 0:
                    see[i] = False                           # a row below position 0 sees nothing
                    continue
                for j in branch(self.parent_list[lo:lo + n], i):
                    if length - n + j >= 0:
                        see[i, length - n + j] = True
            see = see.to(self.device) & there[None]
            rows = slice(lo, lo + n)
            for h in range(self.hq):
                q, kh, vh = self.q[rows, h].double(), k[:, h // group], v[:, h // group]
                s = torch.where(see, (q @ kh.t()) * scale, torch.full_like(see, -torch.inf, dtype=torch.float64))
                z = torch.logsumexp(s, -1)
                p = torch.where(see, torch.exp(s - torch.where(z == -torch.inf, torch.zeros_like(z), z)[:, None]), torch.zeros_like(s))
                vh = torch.where(there[:, None], vh, torch.zeros_like(vh))
                out[rows, h], mass[rows, h], lse[h, rows] = p @ vh, p @ vh.abs(), z
                size[h, rows] = (torch.where(see, q.abs() @ kh.abs().t(), torch.zeros_like(s)) * scale).amax(-1)
        return out, lse, mass, size
