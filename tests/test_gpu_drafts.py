"""GPU: drafted tokens checked against the target's probabilities; the answers are whole numbers and have to be those of the rule in 64 bits."""
import math

import pytest
import torch

from baselinebenchmark_b200 import verify_drafts
from tests.tree_util import random_parents

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _clean(x):
    x = x.double()
    return torch.where((x > 0) & (x < math.inf), x, torch.zeros_like(x))


def rule(target, draft, tokens, news, accept, sample, most, parents=None):
    """The rule of include/moba_b200.h, sequence by sequence on the CPU."""
    paths, tokens_next, lo, v = [], [], 0, target.shape[1]
    for b, n in enumerate(news):
        up = [i - 1 for i in range(n)] if parents is None else parents[lo:lo + n]
        n_seen, at, path, end = min(n, most), 0, [0], n == 0
        if end:
            paths.append([])
            tokens_next.append(-1)
            continue
        while not end:
            t, mass, end = _clean(target[lo + at]), 1.0, True
            q = _clean(draft[lo + at]) if draft is not None else None
            for c in [c for c in range(at + 1, n_seen) if up[c] == at]:
                x = tokens[lo + c]
                have = float(t[x]) if 0 <= x < v else 0.0
                drawn = 1.0 if q is None else float(q[x]) if 0 <= x < v else 0.0
                if have > 0 and accept[lo + c] * mass * drawn < have:
                    at, end = c, False
                    path.append(c)
                    break
                if q is None:
                    mass -= have
                    if 0 <= x < v:
                        t[x] = 0.0
                else:
                    t = ((t / mass if mass > 0 else torch.zeros_like(t)) - q).clamp(min=0)
                    mass = float(t.sum())
        if float(t.sum()) <= 0:
            t = _clean(target[lo + at])
        if float(t.sum()) <= 0:
            tokens_next.append(-1)
        else:
            ends = t.cumsum(0)
            over = torch.nonzero((ends > sample[b] * ends[-1]) & (t > 0))
            tokens_next.append(int(over[0]) if over.numel() else int(torch.nonzero(t > 0)[-1]))
        paths.append(path)
        lo += n
    return ([p + [-1] * (most - len(p)) for p in paths], [len(p) for p in paths], tokens_next)


class Drafts:
    """Sequences with `news` rows; distributions over v tokens of which a handful have most."""

    def __init__(self, news, v, dtype, spread=None, draft=True, seed=0, near=0.5, bits=64):
        g = torch.Generator().manual_seed(seed)
        self.news, rows = news, sum(news)
        self.parents = None if spread is None else random_parents(news, spread, seed)
        x = 2.5 * torch.randn(rows, v, generator=g)
        self.target = torch.softmax(x, -1).to(dtype)
        p = torch.softmax(x + near * torch.randn(rows, v, generator=g), -1)
        self.draft = p.to(dtype) if draft else None
        up = self.parents or [i - 1 for n in news for i in range(n)]
        self.tokens, lo, seen = [], 0, {}
        for n in news:
            for i in range(n):
                if up[lo + i] < 0:
                    self.tokens.append(0)
                    continue
                at = lo + up[lo + i]
                if draft:
                    self.tokens.append(int(torch.multinomial(p[at], 1, generator=g)))
                else:
                    seen[at] = seen.get(at, -1) + 1
                    self.tokens.append(int(p[at].topk(min(seen[at] + 1, v)).indices[-1]))
            lo += n
        self.accept, self.sample = torch.rand(rows, generator=g), torch.rand(len(news), generator=g)
        self.bits = bits

    def check(self, most=None, target=None, draft=None, **kw):
        most = max(max(self.news), 1) if most is None else most
        cu = _i32([0] + [sum(self.news[:i + 1]) for i in range(len(self.news))])
        tokens = torch.tensor(self.tokens, dtype=torch.int64 if self.bits == 64 else torch.int32, device="cuda")
        got = verify_drafts(self.target.cuda() if target is None else target, draft if draft is not None else self.draft.cuda() if self.draft is not None else None,
                            tokens, cu, self.accept.cuda(), self.sample.cuda(), most,
                            parents=_i32(self.parents) if self.parents is not None else None)
        want = rule(self.target, self.draft, self.tokens, self.news, self.accept.double().tolist(), self.sample.double().tolist(), most, self.parents)
        assert got[2].dtype == tokens.dtype
        for x, y in zip(got, want):
            assert x.tolist() == y
        return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [1, 7, 129, 1000, 4097, 33000])
@pytest.mark.parametrize("draft", [True, False])
def test_chains(dtype, v, draft):
    d = Drafts([6, 1, 0, 3, 12], v, dtype, draft=draft, seed=v, near=0.3 if v < 1000 else 0.1)
    d.check()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("spread,seed", [(2, 1), (6, 2), (40, 3), (40, 4)])
def test_trees(dtype, draft, spread, seed):
    """Several siblings, the same token among them, tried one after another against what is left."""
    d = Drafts([40, 17, 2, 1, 64], 900, dtype, spread=spread, draft=draft, seed=seed, near=1.5, bits=32)
    d.check()


@pytest.mark.parametrize("draft", [True, False])
def test_nothing_is_accepted_and_everything(draft):
    for near, force in ((0.2, 0.0), (3.0, 1.0 - 2.0 ** -24)):
        d = Drafts([9, 30], 500, torch.float32, spread=3, draft=draft, near=near, seed=5)
        d.accept.fill_(force)
        _, count, _ = d.check()
        assert (min(count) > 1) == (force == 0.0) or force > 0


@pytest.mark.parametrize("u", [0.0, 0.5, 1.0 - 2.0 ** -24, 1.0, -3.0, math.nan])
def test_borders_of_the_sample(u):
    """Probabilities whose sums are exact; a number from 1 on, and one that is none, take the last token that has any probability."""
    d = Drafts([1, 1, 1], 64, torch.float32, seed=1)
    d.target = torch.zeros(3, 64)
    d.target[0, 5], d.target[0, 9] = 0.5, 0.5
    d.target[1, 63] = 1.0
    d.target[2, ::2] = 2.0 ** -5
    d.sample.fill_(u)
    want = d.check()[2]
    assert want[1] == 63 and want[0] == (9 if not u < 0.5 else 5) and want[2] == (62 if not u < 1 else {0.0: 0, 0.5: 32, -3.0: 0}.get(u, 62))


@pytest.mark.parametrize("draft", [True, False])
def test_values_that_are_no_probabilities(draft):
    d = Drafts([5, 5, 4], 300, torch.float32, spread=3, draft=draft, seed=6, near=1.0)
    g = torch.Generator().manual_seed(1)
    for x in (d.target, d.draft):
        if x is not None:
            where = torch.rand(x.shape, generator=g)
            x[where < 0.1], x[where > 0.95], x[(where > 0.5) & (where < 0.55)] = -1.0, math.nan, math.inf
    d.tokens[1], d.tokens[6] = -5, 300                       # outside the vocabulary
    d.check()
    d.target[10:].zero_()                                    # a sequence with no probabilities at all
    assert d.check()[2][2] == -1


def test_nothing_left():
    """A draft that covers the target everywhere, and siblings that take all of it: the token comes from the whole row."""
    d = Drafts([3, 3], 8, torch.float32, spread=3, seed=3)
    d.parents = [-1, 0, 0] * 2
    d.target = torch.full((6, 8), 0.125)
    d.draft = torch.full((6, 8), 0.5)
    d.accept.fill_(0.9)
    assert d.check()[1] == [1, 1]
    d.draft = None
    d.target = torch.zeros(6, 8)
    d.target[:, 2] = d.target[:, 4] = 0.5
    d.tokens, d.accept = [0, 2, 4] * 2, torch.tensor([0.0, 0.5, 1.0] * 2)
    assert d.check()[1] == [1, 1] and all(x in (2, 4) for x in d.check()[2])


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_addresses(draft, dtype):
    """Rows that are parts of wider ones and begin anywhere."""
    for v, off in ((1001, 1), (1000, 3), (2048, 4), (2048, 0)):
        d = Drafts([4, 9], v, dtype, spread=4, draft=draft, seed=v + off, near=1.0)
        wide = torch.full((13, v + 11), math.nan, dtype=dtype, device="cuda")
        wide[:, off:off + v] = d.target.cuda()
        wide_q = torch.full((13, v + 24), math.nan, dtype=dtype, device="cuda")
        if draft:
            wide_q[:, 8:8 + v] = d.draft.cuda()
        d.check(target=wide[:, off:off + v], draft=wide_q[:, 8:8 + v] if draft else None)


def test_rows_beyond_the_most():
    d = Drafts([30, 5, 12], 200, torch.float32, spread=4, seed=8, near=0.2)
    for most in (1, 2, 11, 40):
        d.check(most=most)


def test_long_chains_and_many_sequences():
    d = Drafts([1024, 3], 40, torch.float32, near=0.0, seed=9)
    d.accept[:1000] = 0.0
    assert d.check()[1][0] > 900
    d = Drafts([2] * 700, 333, torch.float16, seed=10)
    d.check()


def test_a_wide_vocabulary():
    for dtype, draft in ((torch.float32, True), (torch.bfloat16, False)):
        d = Drafts([3, 2], 600011, dtype, spread=2, draft=draft, seed=11, near=0.5)
        d.check()


def test_the_widest_vocabulary_and_many_sequences():
    """All rows have the same distribution, over 2**22 tokens; given tokens, rejected one after another."""
    v, n = 2 ** 22, 600
    g = torch.Generator(device="cuda").manual_seed(16)
    row = torch.rand(v, device="cuda", generator=g)
    row /= row.sum()
    sample = torch.rand(n, device="cuda", generator=g)
    tokens = torch.tensor([0, 5, v - 1, 70], device="cuda").repeat(n)
    cu = torch.arange(0, 4 * n + 1, 4, dtype=torch.int32, device="cuda")
    path, count, after = verify_drafts(row.expand(4 * n, v), None, tokens, cu, torch.ones(4 * n, device="cuda"), sample, 4, parents=_i32([-1, 0, 0, 0]).repeat(n))
    assert (count == 1).all() and (path[:, 0] == 0).all() and (path[:, 1:] == -1).all()
    left = row.double()
    left[[5, v - 1, 70]] = 0.0
    ends = left.cumsum(0)
    assert torch.equal(after, torch.searchsorted(ends, sample.double() * ends[-1], right=True))


def test_captured_and_on_two_streams():
    a, b = Drafts([5, 4], 5000, torch.float32, seed=12, spread=2), Drafts([5, 4], 5000, torch.float32, seed=13, spread=3)
    tensors = lambda d: [d.target.cuda(), d.draft.cuda(), torch.tensor(d.tokens, device="cuda"), d.accept.cuda(), d.sample.cuda(), _i32(d.parents)]  # noqa: E731
    held, cu = tensors(a), _i32([0, 5, 9])
    call = lambda t: verify_drafts(t[0], t[1], t[2], cu, t[3], t[4], 5, parents=t[5])  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = call(held)
    torch.cuda.current_stream().wait_stream(stream)
    for d in (b, a):
        for x, y in zip(held, tensors(d)):
            x.copy_(y)
        graph.replay()
        want = rule(d.target, d.draft, d.tokens, d.news, d.accept.double().tolist(), d.sample.double().tolist(), 5, d.parents)
        assert [x.tolist() for x in got] == list(want)
    streams, out = [torch.cuda.Stream() for _ in range(3)], []
    sets = [tensors(d) for d in (a, b, a)]
    for s, t in zip(streams, sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out.append(call(t))
    torch.cuda.synchronize()
    for d, o in zip((a, b, a), out):
        want = rule(d.target, d.draft, d.tokens, d.news, d.accept.double().tolist(), d.sample.double().tolist(), 5, d.parents)
        assert [x.tolist() for x in o] == list(want)


def test_the_tokens_are_distributed_as_the_targets():
    """100000 sequences with two drafted siblings each: token after token, the target's probabilities to 5 standard deviations."""
    n, v = 100000, 6
    g = torch.Generator(device="cuda").manual_seed(14)
    p = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.05, 0.0], device="cuda")
    q = torch.tensor([0.1, 0.2, 0.3, 0.1, 0.2, 0.1], device="cuda")
    target, draft = p.expand(3 * n, v).contiguous(), q.expand(3 * n, v).contiguous()
    drawn = torch.multinomial(q, 3 * n, replacement=True, generator=g)
    rand = lambda k: torch.rand(k, device="cuda", generator=g)  # noqa: E731
    for with_draft in (True, False):
        tokens = drawn if with_draft else torch.tensor([0, 2, 0], device="cuda").repeat(n)
        cu = torch.arange(0, 3 * n + 1, 3, dtype=torch.int32, device="cuda")
        path, count, after = verify_drafts(target, draft if with_draft else None, tokens, cu, rand(3 * n), rand(n), 3,
                                           parents=_i32([-1, 0, 0]).repeat(n))
        first = torch.where(count > 1, tokens.view(n, 3).gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], after)
        share = torch.bincount(first, minlength=v).double() / n
        assert ((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / n).sqrt() + 1e-9).all()
        behind = after[count > 1]                             # and the token behind an accepted one
        share = torch.bincount(behind, minlength=v).double() / behind.numel()
        assert ((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / behind.numel()).sqrt() + 1e-9).all()


def test_refusals():
    d = Drafts([3, 2], 20, torch.float32, spread=2, seed=15)
    cu, tokens = _i32([0, 3, 5]), torch.tensor(d.tokens, device="cuda")
    base = dict(target=d.target.cuda(), draft=d.draft.cuda(), tokens=tokens, cu_seqlens=cu, accept=d.accept.cuda(), sample=d.sample.cuda(), max_new=3)
    for error, kw in ((ValueError, dict(target=base["target"][0])), (TypeError, dict(target=base["target"].double())), (ValueError, dict(draft=base["draft"][:2])),
                      (TypeError, dict(draft=base["draft"].half())), (ValueError, dict(tokens=tokens[:2])), (TypeError, dict(tokens=tokens.short())),
                      (TypeError, dict(cu_seqlens=cu.long())), (ValueError, dict(cu_seqlens=cu[:1])), (TypeError, dict(accept=base["accept"].half())),
                      (ValueError, dict(sample=base["accept"])), (ValueError, dict(max_new=0)), (NotImplementedError, dict(max_new=1025)),
                      (NotImplementedError, dict(target=base["target"].t().contiguous().t())), (TypeError, dict(accept=d.accept)),
                      (ValueError, dict(parents=_i32([0])), ), (TypeError, dict(parents=torch.zeros(5, device="cuda"))),
                      (NotImplementedError, dict(target=base["target"].clone().requires_grad_()))):
        with pytest.raises(error):
            verify_drafts(**{**base, **kw})
    with torch.no_grad():
        verify_drafts(**{**base, "target": base["target"].clone().requires_grad_()})
    with torch.inference_mode():
        path, count, after = verify_drafts(**base)
    assert path.shape == (2, 3) and count.shape == after.shape == (2,)
    path, count, after = verify_drafts(**{**base, "target": base["target"][:0], "draft": None, "tokens": tokens[:0], "accept": base["accept"][:0]})
    assert (path == -1).all() and count.tolist() == [0, 0] and after.tolist() == [-1, -1]
