"""GPU: the paged cache over values of unusual sizes, for the kernel for few rows (tiles of 8 and of 16) and the one for many."""
import math

import pytest
import torch

from baselinebenchmark_b200 import PagedKV, paged_attention, paged_load
from tests.paged_util import Batch

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, FP16 = torch.bfloat16, torch.float16
#: `max_new` for tiles of 8 rows, of 16, and for the kernel for many rows, with groups of four query heads
KERNELS = [1, 4, 4096]
#: rows, pages
STORES = [(BF16, E4M3), (BF16, INT8), (FP16, E4M3), (FP16, INT8)]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _attend(b, kernel):
    b.fill()
    b.check(*paged_attention(b.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales))


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype,store", STORES)
def test_two_keys_with_a_channel_each(dtype, store, kernel):
    """Equal scores, V rows [2^15, 0, ..] and [0, 2^-10, ..]: the second channel is 2^-11, however much larger the other row is."""
    cache = PagedKV(1, 16, 1, 64, dtype, store)
    k, v = torch.zeros(2, 1, 64), torch.zeros(2, 1, 64)
    k[:, 0, 0] = 1
    v[0, 0, 0], v[1, 0, 1] = 2.0 ** 15, 2.0 ** -10
    where = (_i32([[0]]), _i32([0, 2]), _i32([2]))
    cache.store(k.to(dtype).cuda(), v.to(dtype).cuda(), *where)
    out = cache.attend(torch.ones(1, 4, 64, dtype=dtype, device="cuda"), where[0], _i32([0, 1]), where[2], kernel).double()
    want = torch.zeros(64, dtype=torch.float64, device="cuda")
    want[0], want[1] = 2.0 ** 14, 2.0 ** -11
    # the weights are halves; a cubic's 1e-4 in numerator and denominator, a rounding of P and one of the output
    assert ((out - want).abs() <= want * (2e-4 + torch.finfo(dtype).eps)).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype,store", STORES)
@pytest.mark.parametrize("size", [1.0, 2.0 ** -10])
def test_v_rows_of_zeros(dtype, store, size, kernel):
    """Rows of V that are zeros take their share of the weights and nothing else, also the one with most of it (a first token that is attended
    to and adds nothing): 2^10 and 2^24 times the others', the former where weights are fp16, which holds the others' then."""
    b = Batch([(1, 500), (3, 777), (2, 40)], 8, 2, 128, 16, dtype, store, seed=70, q_scale=0.25)
    gap = 7.0 if dtype == FP16 else 17.0
    for i, (k, v) in enumerate(b.hist):
        v *= size
        v[5::9] = 0
        v[0] = 0
        # the first key: the sum of a kv head's queries, stretched until each of them scores `gap` or more above its average
        rows = b.q[b.cu_list[i]:b.cu_list[i + 1]].cpu().float().unflatten(1, (2, 4))
        mean = rows.mean((0, 2))
        least = (rows * mean[None, :, None]).sum(-1).amin((0, 2)) / 128 ** 0.5
        good = least > 0.05
        k[0] = torch.where(good[:, None], mean * (gap / least.clamp(min=0.05))[:, None], k[0].float()).to(dtype)
    _attend(b, kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype,store", STORES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_v_rows_with_one_large_channel(dtype, store, dim, kernel):
    """Every seventh row of V has one element, which no other row has: its power of two is far above the others', and they alone make
    all other channels."""
    b = Batch([(1, 400), (4, 300), (2, 33)], 8, 2, dim, 32, dtype, store, seed=71 + dim, q_scale=0.5)
    for _, v in b.hist:
        big = v[::7]
        v[:, :, 5] = 0
        big[:] = 0
        big[:, :, 5] = 2.0 ** 15 if dtype == FP16 else 2.0 ** 30
        v[1::7] *= 2.0 ** -9 if dtype == FP16 else 2.0 ** -20
    _attend(b, kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("store", [E4M3, INT8])
def test_scores_far_apart_and_a_channel_each(store, kernel):
    """bfloat16 weights have the range of fp32: keys 2^-30 and 2^-60 of the largest weight still make the channels that they alone have."""
    cache = PagedKV(8, 16, 1, 128, BF16, store)
    n = 100
    k, v = torch.zeros(n, 1, 128), torch.zeros(n, 1, 128)
    score = torch.zeros(n)
    score[10:40], score[40:90], score[90:] = -20.0, -41.0, -60.0     # natural log
    k[:, 0, 0] = score
    v[:10, 0, :32], v[10:40, 0, 32:64], v[40:90, 0, 64:96], v[90:, 0, 96:] = 1.0, 1.0, 2.0 ** 20, 2.0 ** -20
    where = (_i32([[3, 1, 0, 7, 2, 6, 5]]), _i32([0, n]), _i32([n]))
    cache.store(k.to(BF16).cuda(), v.to(BF16).cuda(), *where)
    q = torch.zeros(1, 4, 128, dtype=BF16, device="cuda")
    q[..., 0] = 1.0
    k64 = cache.load(*where, n)[0].double()[:, 0, 0]
    p = torch.softmax(k64, 0)
    v64 = cache.load(*where, n)[1].double()[:, 0]
    want = p @ v64
    out = cache.attend(q, where[0], _i32([0, 1]), where[2], kernel, scale=1.0).double()
    # a score's exponential is off by 2^-24 of the score (60 at most) and by 1e-4; one rounding of P, one of the output
    tol = want * (2 * (1e-4 + 60 * 2.0 ** -23) + 2.0 ** -8 + 2.0 ** -8)
    assert (want > 0).all() and ((out - want).abs() <= tol).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype,store", STORES)
def test_zeros_alone(dtype, store, kernel):
    """Nothing but zeros in V, and a pool that nothing was ever written to."""
    b = Batch([(1, 100), (2, 50)], 8, 2, 64, 16, dtype, store, seed=72)
    for _, v in b.hist:
        v.zero_()
    _attend(b, kernel)
    cache = PagedKV(4, 16, 2, 64, dtype, store)
    q = torch.ones(1, 8, 64, dtype=dtype, device="cuda")
    out, lse = cache.attend(q, _i32([[0, 1, 2, 3]]), _i32([0, 1]), _i32([60]), kernel, return_lse=True)
    assert (out == 0).all() and (lse - math.log(60)).abs().max() < 1e-3


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("store", [E4M3, INT8])
@pytest.mark.parametrize("big,small", [(2.0 ** 14, 2.0 ** -20), (2.0 ** 40, 2.0 ** -1), (2.0 ** 110, 2.0 ** -10), (2.0 ** -70, 2.0 ** -100)])
def test_queries_with_a_channel_for_some_keys(store, big, small, kernel):
    """A query's largest element meets zeros in every key: what the others, however much smaller, make of the keys decides."""
    b = Batch([(1, 300), (4, 200)], 8, 2, 128, 16, BF16, store, seed=73)
    for k, _ in b.hist:
        k[:, :, 9] = 0
        k /= small
    b.q *= small
    b.q[:, :, 9] = big
    _attend(b, kernel)


@pytest.mark.parametrize("store", [E4M3, INT8])
@pytest.mark.parametrize("kernel", KERNELS)
def test_float16_queries_over_rows_written_from_bfloat16(store, kernel):
    """The rows count as `paged_load` gives them in the queries' type: rounded to it, infinities above its range, whichever kernel runs."""
    seqs = [(1, 300), (4, 200), (2, 100)]
    b = Batch(seqs, 8, 2, 64, 16, BF16, store, seed=74)
    for k, v in b.hist:
        k[:, :, 3:] *= 2.0 ** -3
        k[::5] *= 2.0 ** -12
        v[1::4] *= 2.0 ** -11
        v[2::4, :, 10:20] *= 2.0 ** 12                       # up to 2^14 or so: within fp16
    b.fill()
    k, v = b.hist[1]
    k[30, 0, 7], v[77, 1, 5], v[78, 1, 6], v[79, 1, 6] = 2.0 ** 20, 1e5, -3e5, 3.0e38
    b.fill()
    half = Batch(seqs, 8, 2, 64, 16, FP16, store, seed=74)
    got, lse = paged_attention(half.q, b.k, b.v, *b.where, kernel, return_lse=True, **b.scales)
    # what the rows are in fp16
    whole = torch.cat([torch.tensor([0]), torch.tensor([n for _, n in seqs]).cumsum(0)]).tolist()
    rows = [x.cpu() for x in paged_load(b.k, b.v, b.table, _i32(whole), b.lens, whole[-1], dtype=FP16, **b.scales)]
    assert torch.isinf(rows[0]).sum() == 1 and torch.isinf(rows[1]).sum() == 3
    bad = torch.isinf(rows[1]).flatten().nonzero()
    half.hist = [tuple(x[whole[i]:whole[i + 1]] for x in rows) for i in range(3)]
    half.store = FP16
    # an infinite key element: -inf or +inf, as the query's element has it; +inf makes NaN.  An infinite value makes its channel infinite or NaN.
    own = slice(1, 5)
    hit = half.q[own, :4, 7] > 0
    assert torch.equal(torch.isnan(got[own, :4]).all(-1), hit) and torch.equal(torch.isnan(lse[:4, own].t()), hit)
    assert (~torch.isfinite(got[own, 4:, 5])).all() and (~torch.isfinite(got[own, 4:, 6])).all()
    # everything else as the formula has it, with the key that scored -inf out of it
    half.hist[1][0][torch.isinf(half.hist[1][0])] = 0
    half.hist[1][1][torch.isinf(half.hist[1][1])] = 0
    out, ref, mass, size = half.attention()
    fine = torch.ones(half.rows, 8, 64, dtype=torch.bool, device="cuda")
    fine[own, :4] = False
    fine[own, 4:, 5:7] = False
    got = torch.where(fine, got, out.to(FP16))
    half.check(got, None, (out, ref, mass, size))
    assert len(bad) == 3


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("store", [E4M3, INT8])
def test_float16_rows_up_to_the_largest(store, kernel):
    """fp16 rows up to 65504, whose codes come near the border of the type."""
    b = Batch([(1, 300), (3, 100)], 8, 2, 128, 32, FP16, store, seed=75)
    for k, v in b.hist:
        k[::3, :, 4] = 60000.0
        k[1::3, :, 4] = -65504.0
        v[::4] = (v[::4].float() * 3e4).clamp(-65504, 65504).to(FP16)
    b.q[:, :, 4] *= 2.0 ** -14
    _attend(b, kernel)
