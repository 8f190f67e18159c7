"""GPU: rotary positions against the formula in 64 bits, and their derivatives.

Bounds: the reduced angle is rounded to 24 bits, half a step of at most 2^-24 half turns (2^-25 pi); the frequency's 2^-65 turns a position add 2^-34 at
most; sine and cosine have 2 units in the last place, 2^-23, the factor and each of two products and their sum 2^-24.  So u cos - v sin is off by
(|u| + |v|) m (2^-25 pi + 2^-34 + 2^-23 + 4 * 2^-24) < (|u| + |v|) m 2^-21, and the rounding to 16 bits adds half a step of the result."""
import math

import pytest
import torch

from baselinebenchmark_b200 import RotaryTable, parallel_moba, rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def turned(x, positions, f, interleaved, magnitude=1.0, inverse=False):
    """float64 (rows turned, |u| + |v| of each element's pair)."""
    d = 2 * f.numel()
    a = positions.double()[:, None] * f.cuda()
    cos, sin = (g(a)[:, None] * magnitude for g in (torch.cos, torch.sin))
    if inverse:
        sin = -sin
    y, size = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    one, two = (slice(0, d, 2), slice(1, d, 2)) if interleaved else (slice(0, d // 2), slice(d // 2, d))
    u, v = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = u * cos - v * sin, u * sin + v * cos
    size[..., one] = size[..., two] = (u.abs() + v.abs()) * magnitude
    none = (positions < 0)[:, None, None]
    return torch.where(none, x.double(), y), torch.where(none, torch.zeros_like(size), size)


def close(got, want, size):
    half = torch.finfo(got.dtype).eps / 2
    tol = size * 2.0 ** -21 * (1 + half) + half * want.abs() + torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    assert ((got.double() - want).abs() <= tol).all()


def _rows(tokens, heads, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(tokens, heads, dim, device="cuda", dtype=dtype, generator=g)


def _positions(tokens, far, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(far, (tokens,), device="cuda", generator=g).int()


@pytest.mark.parametrize("tokens,hq,hkv,dim,turn", [(1, 1, 1, 64, 64), (3, 5, 1, 96, 96), (70, 32, 8, 128, 128), (9, 4, 2, 256, 256), (33, 6, 3, 128, 64),
                                                    (12, 3, 3, 96, 24), (5, 7, 1, 64, 2), (40, 2, 2, 256, 90), (6, 12, 4, 128, 126), (1500, 8, 2, 64, 16),
                                                    (2000, 40, 8, 128, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_turned_rows(tokens, hq, hkv, dim, turn, interleaved, dtype):
    q, k, pos = _rows(tokens, hq, dim, dtype), _rows(tokens, hkv, dim, dtype, 2), _positions(tokens, 5000)
    if tokens > 2:
        pos[1], pos[2] = -1, 0
    f = rotary_frequencies(turn)
    for magnitude in (1.0, 1.2772588722):
        table = RotaryTable(f, interleaved=interleaved, magnitude=magnitude)
        got = rotary(q, k, pos, table)
        for x, y in ((q, got[0]), (k, got[1])):
            assert y.is_contiguous() and y.dtype == dtype
            close(y, *turned(x, pos, f, interleaved, torch.tensor(magnitude).double().item()))
            assert torch.equal(y[..., turn:], x[..., turn:])
    alone, none = rotary(q, None, pos, table)
    assert none is None and torch.equal(alone, got[0])


@pytest.mark.parametrize("far", [1 << 20, 2 ** 31 - 1])
def test_far_positions(far):
    """Angles of millions of radians; in 64 bits such an angle itself is off by 2^31 * 2^-53."""
    q, pos = _rows(300, 2, 128, torch.float16), _positions(300, far)
    pos[0] = far - 1
    f = rotary_frequencies(128)
    close(rotary(q, None, pos, RotaryTable(f))[0], *turned(q, pos, f, False))


@pytest.mark.parametrize("scaling,kw", [("linear", {}), ("base", {}), ("parts", dict(original=4096)), ("parts", dict(original=8192, fast=4.0))])
def test_scaled_frequencies(scaling, kw):
    q, pos = _rows(64, 4, 128, torch.bfloat16), _positions(64, 100000)
    f = rotary_frequencies(128, 500000.0, scaling=scaling, factor=8.0, **kw)
    close(rotary(q, None, pos, RotaryTable(f, magnitude=1.3))[0], *turned(q, pos, f, False, torch.tensor(1.3).double().item()))


@pytest.mark.parametrize("turn,interleaved", [(128, False), (128, True), (40, False), (6, True)])
def test_in_place_and_strides(turn, interleaved):
    """Views of a fused projection turned where they are; broadcast rows; output into a wider tensor.  What is beside them stays."""
    qkv, pos = _rows(50, 12, 128, torch.bfloat16), _positions(50, 3000)
    pos[7] = -1
    table, before = RotaryTable(rotary_frequencies(turn), interleaved=interleaved), qkv.clone()
    want = rotary(before[:, :6], before[:, 6:9], pos, table)
    wide = torch.full((50, 14, 128), 7.0, dtype=qkv.dtype, device="cuda")
    other = torch.full((3, 50, 128), 7.0, dtype=qkv.dtype, device="cuda").transpose(0, 1)
    got = rotary(qkv[:, :6], qkv[:, 6:9], pos, table, out=(wide[:, 4:10], other))
    assert torch.equal(got[0], want[0]) and torch.equal(other, want[1]) and (wide[:, :4] == 7).all() and (wide[:, 10:] == 7).all()
    version = qkv._version
    q, k = qkv[:, :6], qkv[:, 6:9]
    assert rotary(q, k, pos, table, out=(q, k))[0] is q and qkv._version > version
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 9:], before[:, 9:]) and torch.equal(q[7], before[7, :6])
    row = before[:1, :1].expand(50, 6, 128)
    assert torch.equal(rotary(row, None, pos, table)[0], rotary(row.contiguous(), None, pos, table)[0])
    assert rotary(q[:0], k[:0], pos[:0], table)[0].shape == (0, 6, 128)


@pytest.mark.parametrize("turn,interleaved", [(64, False), (64, True), (12, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients(turn, interleaved, dtype):
    q, k, pos = _rows(21, 4, 64, dtype).requires_grad_(), _rows(21, 2, 64, dtype, 3).requires_grad_(), _positions(21, 900)
    f = rotary_frequencies(turn)
    table = RotaryTable(f, interleaved=interleaved, magnitude=1.25)
    dq, dk = _rows(21, 4, 64, dtype, 4), _rows(21, 2, 64, dtype, 5)
    got = torch.autograd.grad(rotary(q, k, pos, table), (q, k), (dq, dk))
    for g, d in zip(got, (dq, dk)):
        close(g, *turned(d, pos, f, interleaved, 1.25, inverse=True))
    # each alone, and gradients that are broadcast or lie any way
    (only,) = torch.autograd.grad(rotary(q, k, pos, table)[1], k, dk)
    assert torch.equal(only, got[1])
    (only,) = torch.autograd.grad(rotary(q, None, pos, table)[0], q, dq.transpose(0, 2).contiguous().transpose(0, 2))
    assert torch.equal(only, got[0])
    (ones,) = torch.autograd.grad(rotary(q, k, pos, table)[0].sum(), q)
    close(ones, *turned(torch.ones_like(q), pos, f, interleaved, 1.25, inverse=True))
    # a row that all tokens share has the sum of theirs
    shared = _rows(1, 4, 64, dtype).requires_grad_()
    (total,) = torch.autograd.grad(rotary(shared.expand(21, 4, 64), None, pos, table)[0], shared, dq)
    want, size = turned(dq, pos, f, interleaved, 1.25, inverse=True)
    u = torch.finfo(dtype).eps / 2                            # (each row's gradient is rounded, and so is their sum)
    assert ((total.double() - want.sum(0)).abs() <= (want.abs().sum(0) + size.sum(0) * 2.0 ** -20) * 2 * u + 1e-6).all()


def test_gradients_of_one_of_two_and_at_odd_addresses():
    q, k, pos = _rows(9, 4, 64, torch.bfloat16), _rows(9, 2, 64, torch.bfloat16, 3), _positions(9, 900)
    table, f = RotaryTable(rotary_frequencies(64)), rotary_frequencies(64)
    odd = torch.zeros(9 * 2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(9, 2, 64)   # contiguous, 2 bytes behind a vector's boundary
    odd.copy_(_rows(9, 2, 64, torch.bfloat16, 4))
    leaf = k.clone().requires_grad_()
    tq, tk = rotary(q, leaf, pos, table)
    assert tq.requires_grad and tk.requires_grad
    (grad,) = torch.autograd.grad(tk, leaf, odd)
    close(grad, *turned(odd, pos, f, False, inverse=True))


def test_differences_and_second_order():
    """(f(x + h e) - f(x - h e)) / 2h is exact for a linear operator but for the roundings: fp16 rows, h = 1, half a step of each value."""
    q, pos = _rows(4, 1, 64, torch.float16), _positions(4, 50)
    table, d = RotaryTable(rotary_frequencies(64)), _rows(4, 1, 64, torch.float16, 7)
    x = q.clone().requires_grad_()
    (grad,) = torch.autograd.grad(rotary(x, None, pos, table)[0], x, d)
    for j in (0, 5, 31, 32, 63):
        e = torch.zeros_like(q)
        e[..., j] = 1.0
        up, down = (rotary((q + s * e), None, pos, table)[0].double() for s in (1, -1))
        step = ((q + e).double() - (q - e).double())[..., j]
        moved = ((up - down) * d.double()).sum(-1) / step
        # half steps: 2^-11 of two values below 4 (64 dims times |d|), and of the gradient
        tol = (d.double().abs() * 2 * 2.0 ** -11 * 8.0).sum(-1) / step.abs() + 2.0 ** -11 * grad[..., j].double().abs() + 1e-6
        assert ((moved - grad[..., j].double()).abs() <= tol).all()
    # the gradient's gradient is the turn, and the tangent is it too
    y = d.clone().requires_grad_()
    x = q.clone().requires_grad_()
    (g,) = torch.autograd.grad(rotary(x, None, pos, table)[0], x, y, create_graph=True)
    (second,) = torch.autograd.grad(g, y, q)
    assert torch.equal(second, rotary(q, None, pos, table)[0])
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, d)
        turned_dual = rotary(dual, dual, pos, table)
        for out in turned_dual:
            primal, tangent = torch.autograd.forward_ad.unpack_dual(out)
            assert torch.equal(primal, rotary(q, None, pos, table)[0]) and torch.equal(tangent, rotary(d, None, pos, table)[0])


def test_in_front_of_moba():
    """A training step: turned queries and keys through the operator; gradients reach the rows before the turn."""
    lens, table = [300, 212], RotaryTable(rotary_frequencies(128))
    pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
    cu = torch.tensor([0, 300, 512], dtype=torch.int32, device="cuda")
    q, k, v = (_rows(512, h, 128, torch.bfloat16, 20 + i).requires_grad_() for i, h in enumerate((4, 2, 2)))
    d = _rows(512, 4, 128, torch.bfloat16, 30)
    tq, tk = rotary(q, k, pos, table)
    # (of one backward: the operator's dk depends on the order in which rows of a routed list are added)
    grads = torch.autograd.grad(parallel_moba(tq, tk, v, cu, 300, 64, 3), (q, k, v, tq, tk), d)
    close(grads[0], *turned(grads[3], pos, rotary_frequencies(128), False, inverse=True))
    close(grads[1], *turned(grads[4], pos, rotary_frequencies(128), False, inverse=True))


def test_captured_forward_and_backward():
    q, k, pos = _rows(30, 4, 128, torch.bfloat16).requires_grad_(), _rows(30, 2, 128, torch.bfloat16, 2).requires_grad_(), _positions(30, 999)
    table, dq, dk = RotaryTable(rotary_frequencies(128)), _rows(30, 4, 128, torch.bfloat16, 3), _rows(30, 2, 128, torch.bfloat16, 4)
    step = lambda: torch.autograd.grad(rotary(q, k, pos, table), (q, k), (dq, dk))  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = step()
    torch.cuda.current_stream().wait_stream(stream)
    pos.copy_(_positions(30, 5000, 9))
    dq.copy_(_rows(30, 4, 128, torch.bfloat16, 8))
    graph.replay()
    for x, y in zip(got, step()):
        assert torch.equal(x, y)


def test_refusals():
    q, k, pos, table = _rows(3, 2, 64, torch.bfloat16), _rows(3, 1, 64, torch.bfloat16), _positions(3, 9), RotaryTable(rotary_frequencies(64))
    for error, args in ((ValueError, (q[0], k, pos, table)), (ValueError, (q, k[:2], pos, table)), (TypeError, (q, k.half(), pos, table)),
                        (TypeError, (q.float(), k.float(), pos, table)), (ValueError, (q, k, pos[:2], table)), (TypeError, (q, k, pos.long(), table)),
                        (TypeError, (q, k, pos.cpu(), table)), (ValueError, (q, k, pos, RotaryTable(rotary_frequencies(66)))),
                        (TypeError, (q, k, pos, RotaryTable(rotary_frequencies(64), device="cpu"))), (ValueError, (q.cpu(), k, pos, table)),
                        (NotImplementedError, (_rows(3, 2, 80, torch.bfloat16), None, pos, table)),
                        (NotImplementedError, (_rows(3, 64, 64, torch.bfloat16).transpose(1, 2), None, pos, table))):
        with pytest.raises(error):
            rotary(*args)
    with pytest.raises(ValueError, match="each of q and k"):
        rotary(q, k, pos, table, out=(q, None))
    with pytest.raises(ValueError, match="out"):
        rotary(q, k, pos, table, out=(q[:2], k))
    with pytest.raises(RuntimeError, match="error -1"):                   # rows on one another
        rotary(q, None, pos, table, out=(q[:1].expand(3, 2, 64), None))
    other = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="error -1"):                   # where the rows are, but not the same way
        rotary(other[:, ::2], None, pos, table, out=(other[:, :2], None))
    with pytest.raises(RuntimeError, match="error -6"):
        rotary(torch.zeros(3 * 130, dtype=torch.bfloat16, device="cuda").as_strided((3, 2, 64), (130, 65, 1)), None, pos, table)
    leaf = q.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="follow"):
        rotary(leaf, None, pos, table, out=(q, None))
    with torch.no_grad():
        with pytest.raises(NotImplementedError):
            rotary(q, None, pos, table, out=(leaf, None))
        rotary(leaf, None, pos, table)
    assert math.isfinite(table.magnitude)
