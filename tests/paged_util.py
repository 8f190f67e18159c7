"""Shared by the tests of the paged cache: batches with their page tables, and plain implementations in 64 bits."""
import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
#: the largest finite value that a code may stand for, by (pages, rows)
MOST = {(torch.float8_e4m3fn, torch.bfloat16): 240.0 * 2.0 ** 120, (torch.int8, torch.bfloat16): 63.0 * 2.0 ** 122,
        (torch.float8_e4m3fn, torch.float16): 240.0 * 2.0 ** 8, (torch.int8, torch.float16): 63.0 * 2.0 ** 10}


def two(e):
    """2^e in float64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantise(x, store):
    """(codes as float64, bytes) of rows x [..., D]: the rule of include/moba_b200.h."""
    y = x.double()
    amax = y.abs().amax(-1)
    # the least e with top * 2^e >= amax: amax / top is 2^(e - 1) < .. <= 2^e.  Both are numbers of at most 11 bits: in float64 the quotient is
    # a power of two when it is one, and nowhere near one otherwise.
    m, e = torch.frexp(torch.where(torch.isfinite(amax), amax, torch.zeros_like(amax)) / TOP[store])
    e = torch.where(m == 0.5, e - 1, e).long().clamp(min=-96)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    bad = ~torch.isfinite(y).all(-1)
    e = torch.where(bad, torch.full_like(e, 128), e)
    y = torch.where(bad[..., None], torch.zeros_like(y), y).clamp(-MOST[store, x.dtype], MOST[store, x.dtype])
    y = y / two(e)[..., None]
    if store == torch.int8:
        codes = y.round()                                    # halves to even
    else:
        step = two(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
        codes = (y / step).round() * step
    return codes, (e + 127).to(torch.uint8)


def values(codes, byte):
    """What codes stand for: float64; a byte of 255 makes NaN."""
    v = codes.double() * two(byte.int() - 127)[..., None]
    return torch.where((byte == 255)[..., None], torch.full_like(v, math.nan), v)


class Batch:
    """A batch of sequences [(new, length)], their table over a shuffled pool and the pool itself.

    Slots that no sequence owns, and slots behind a sequence's end, hold NaN.  `layout`: "heads" (head-major pages) or "tokens"."""

    def __init__(self, seqs, hq, hkv, dim, page, dtype=torch.bfloat16, store=None, seed=0, layout="heads", device="cuda",
                 spare=3, missing=(), scale=1.0, q_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.hq, self.hkv, self.dim, self.page, self.dtype = seqs, hq, hkv, dim, page, dtype
        self.store = dtype if store is None else store
        need = [-(-max(n, 0) // page) for _, n in seqs]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        per = max(max(need), 1) + 1
        table = torch.full((len(seqs), per), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = order.pop()
        # a page number that is none, where a sequence has none
        table[:, -1] = torch.tensor([(-7, self.pages, 2 ** 31 - 1)[b % 3] for b in range(len(seqs))], dtype=torch.int32)
        for b, i in missing:
            table[b, i] = -1 if b % 2 else self.pages + 5
        cu = [0]
        for n, _ in seqs:
            cu.append(cu[-1] + n)
        self.rows, self.max_new = cu[-1], max(max(n for n, _ in seqs), 1)
        self.cu_list, self.table_list = cu, table.tolist()
        rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.hist = []                                       # K and V rows [len, Hkv, D] of each sequence, the new ones last
        for _, n in seqs:
            k = rand(max(n, 0), hkv, dim) * scale + 0.25 * rand(1, hkv, dim)
            self.hist.append((k.to(dtype), (rand(max(n, 0), hkv, dim) * scale).to(dtype)))
        self.q = (rand(self.rows, hq, dim) * q_scale).to(dtype).to(device)
        new = [[], []]
        for (n, length), kv in zip(seqs, self.hist):
            for i in range(2):
                old = max(n - max(length, 0), 0)             # rows at positions below zero
                new[i].append(torch.cat([rand(old, hkv, dim).to(dtype), kv[i][max(length, 0) - (n - old):]]) if n else kv[i][:0])
        self.k_new, self.v_new = (torch.cat(x).to(device) for x in new)
        self.table, self.cu = table.to(device), torch.tensor(cu, dtype=torch.int32, device=device)
        self.lens = torch.tensor([n for _, n in seqs], dtype=torch.int32, device=device)
        self.layout, self.device = layout, device
        self.k, self.ks = self._pool()
        self.v, self.vs = self._pool()

    def _pool(self):
        shape = (self.pages, self.hkv, self.page, self.dim) if self.layout == "heads" else (self.pages, self.page, self.hkv, self.dim)
        if self.store == self.dtype:
            x, s = torch.full(shape, math.nan, dtype=self.dtype, device=self.device), None
        else:
            x = torch.full(shape, 0x7f, dtype=torch.int8, device=self.device).view(self.store)
            s = torch.full((self.pages, self.hkv, self.page), 255, dtype=torch.uint8, device=self.device)
        return (x.transpose(1, 2) if self.layout == "heads" else x), s

    def page_of(self, b, pos):
        i = pos // self.page
        if pos < 0 or i >= len(self.table_list[b]):
            return -1
        p = self.table_list[b][i]
        return p if 0 <= p < self.pages else -1

    def fill(self, new=True):
        """Puts the history into the pools with plain torch; without `new` only the tokens before the packed ones."""
        for (n, length), kv, b in zip(self.seqs, self.hist, range(len(self.seqs))):
            for i in range(0, max(length if new else length - n, 0), self.page):
                p = self.page_of(b, i)
                if p < 0:
                    continue
                stop = min(i + self.page, length if new else length - n)
                for pool, scales, rows in ((self.k, self.ks, kv[0]), (self.v, self.vs, kv[1])):
                    x = rows[i:stop].to(self.device)
                    if scales is None:
                        pool[p, :stop - i] = x
                    else:
                        codes, byte = quantise(x, self.store)
                        pool.view(torch.int8)[p, :stop - i] = codes.to(torch.float32).to(self.store).view(torch.int8)
                        scales[p].t()[:stop - i] = byte

    @property
    def scales(self):
        return {"k_scales": self.ks, "v_scales": self.vs}

    @property
    def where(self):
        return self.table, self.cu, self.lens

    def stored(self, b, which):
        """float64 rows [len, Hkv, D] that sequence b's pages stand for, and which of them are there."""
        x = self.hist[b][which].to(self.device)
        v = x.double() if self.store == self.dtype else values(*quantise(x, self.store))
        there = torch.tensor([self.page_of(b, i) >= 0 for i in range(x.shape[0])], dtype=torch.bool, device=self.device)
        return v, there

    def attention(self, scale=None):
        """float64 (out [T, Hq, D], lse [Hq, T], weight [T, Hq, D] = sum p |v|, size of the scores [Hq, T])."""
        scale = self.dim ** -0.5 if scale is None else scale
        out = torch.zeros(self.rows, self.hq, self.dim, dtype=torch.float64, device=self.device)
        mass, lse = torch.zeros_like(out), torch.full((self.hq, self.rows), -math.inf, dtype=torch.float64, device=self.device)
        size = torch.zeros_like(lse)
        group = self.hq // self.hkv
        for b, (n, length) in enumerate(self.seqs):
            if n == 0 or length <= 0:
                continue
            (k, there), (v, _) = self.stored(b, 0), self.stored(b, 1)
            rows = slice(self.cu_list[b], self.cu_list[b + 1])
            pos = torch.arange(length - n, length, device=self.device)
            see = (torch.arange(length, device=self.device)[None] <= pos[:, None]) & there[None]
            for h in range(self.hq):
                q = self.q[rows, h].double()
                s = (q @ k[:, h // group].t()) * scale
                s = torch.where(see, s, torch.full_like(s, -math.inf))
                z = torch.logsumexp(s, -1)
                p = torch.where(see, torch.exp(s - torch.where(z == -math.inf, torch.zeros_like(z), z)[:, None]), torch.zeros_like(s))
                vh = torch.where(there[:, None], v[:, h // group], torch.zeros_like(v[:, h // group]))
                out[rows, h], mass[rows, h] = p @ vh, p @ vh.abs()
                lse[h, rows] = z
                size[h, rows] = (torch.where(see, q.abs() @ k[:, h // group].abs().t(), torch.zeros_like(s)) * scale).amax(-1)
        return out, lse, mass, size

    def check(self, got, lse=None, want=None, scale=None):
        """Bounds on every element.  u: half a step of the 16-bit type.  P is rounded once (u of the sum of p |v|) and so is the
        output; a score is off by at most (D + 8) 2^-24 of the sum of |q k| (fp32 products and sums, q's power of two and the
        factor exact to a rounding each), which makes its exponential off by as much, relatively; the exponential itself by 1e-4 (a
        cubic) and the sums over the keys by 2^-24 a key; numerator and denominator each."""
        out, ref, mass, size = self.attention(scale) if want is None else want
        u = torch.finfo(self.dtype).eps / 2
        keys = max((n for _, n in self.seqs), default=1)
        e = 2 * ((self.dim + 8) * 2.0 ** -24 * size + 1e-4 + max(keys, 1) * 2.0 ** -24)
        tol = mass * (u + e.t()[..., None]) + u * out.abs() + torch.finfo(self.dtype).tiny
        d = (got.double() - out).abs()
        assert torch.isfinite(got).all()
        assert (d <= tol).all(), f"largest excess {(d / tol).max().item():.3g} of the bound"
        if lse is not None:
            none = torch.isinf(ref)
            assert torch.equal(lse.double()[none], ref[none])
            assert ((lse.double() - ref)[~none].abs() <= (e + 2.0 ** -22 * ref.abs())[~none]).all()
