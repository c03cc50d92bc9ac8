"""Attention of new rows over the pages where its numbers are at their limits:
weights far below a row's largest, NaN and infinities that the rows see, units
of one kind and the other, calls of fewer rows than their sequences bring."""
import math

import pytest
import torch

from serving_ref import DT, Batch, half_step
from test_chunk_attention_gpu import bound, call

pytestmark = pytest.mark.gpu

TYPES = ["f32", "f16", "bf16"]


def place(B, b, lo, hi, k=None, v=None):
    """Keys and values of positions [lo, hi) of sequence b: scalars, or one number for each position."""
    pages, slot = B.slots(b, lo, hi)
    for pool, x in ((B.k, k), (B.v, v)):
        if x is not None:
            x = torch.as_tensor(x, dtype=torch.float64, device="cuda")
            pool[pages, :, slot] = (x[:, None, None] if x.dim() else x).to(pool.dtype)


def queries(B, heads, value=1.0):
    return torch.full((B.rows, heads * B.hd), value, dtype=DT[B.typ], device="cuda")


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n", [1, 70])  # units of few rows, whose weights have two parts, and of more than 128
def test_many_small_weights_beside_a_large_one(gb, kernels, cuda, typ, n):
    # Position 0 outweighs each of the others by 17 to 20 in the exponent and its value is 0, so the result is what
    # the others' weights of 2e-9 to 4e-8 leave: all of them count. As many units as CTAs, so that none is cut.
    # Beyond the bound of ordinary rows: binary16 holds a weight times 2^7 at least, and a number below its smallest
    # normal one is off by 2^-25 at most, so each of N positions adds 2^-32 of its |v| to the error, and the result
    # is such a number too.
    kv, n_kv = 2000, 148
    B = Batch([(n, kv)], n_kv, 64, 64, typ, 300)
    g = torch.Generator().manual_seed(301)
    k, v = torch.rand(kv, generator=g) * 0.375 - 0.25, 1 + torch.rand(kv, generator=g)
    k[0], v[0] = 2.25, 0.0  # a score of 18 beside scores of -2 to 1
    place(B, 0, 0, kv, k=k, v=v)
    q = queries(B, 2 * n_kv)
    out = torch.zeros_like(q)
    want, mag, big = B.attention(q, 2 * n_kv, 0.125, out)
    call(gb, kernels, B, q, 2 * n_kv, 0.125, out)
    torch.cuda.synchronize()
    tol = bound(typ, 64, kv, want, mag, big) + (kv * 2.0 ** -32 * 2 + 2.0 ** -25 if typ == "f16" else 0)
    assert (tol < 0.2 * want).all()  # the bound tells a result from none
    assert ((out.double() - want).abs() <= tol).all(), float(((out.double() - want).abs() / want).max())


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n", [1, 5, 100])  # joined by a warp a row, and in slices
@pytest.mark.parametrize("kv", [200, 9000])  # one CTA's piece, and pieces of many
def test_a_nan_shows_however_small_its_weight(gb, kernels, cuda, typ, n, kv):
    # position 10 holds NaN in V and weighs 2^-180 of the largest: 0 in float32, and 0 NaN is NaN
    B = Batch([(n, kv), (1, 300)], 1, 64, 16, typ, 310)
    low = 64 if kv < 1000 else kv // 2
    place(B, 0, 0, low, k=-16.0)
    place(B, 0, low, kv, k=0.0)
    place(B, 0, 10, 11, v=math.nan)
    q = queries(B, 4)
    out = torch.zeros_like(q)
    call(gb, kernels, B, q, 4, 0.125, out)
    torch.cuda.synchronize()
    assert out[:n].isnan().all() and out[n:].isfinite().all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n,kv", [(1, 1), (1, 700), (1, 9000), (90, 90), (200, 9000)])
def test_rows_of_scores_minus_infinity(gb, kernels, cuda, typ, n, kv):
    # every score a row sees is -infinity: its softmax is 0 / 0. A row that sees nothing is zeros all the same.
    B = Batch([(n, kv), (3, 2), (1, 300)], 2, 64, 16, typ, 320)
    place(B, 0, 0, kv, k=-math.inf)
    q = queries(B, 8)
    out = torch.full_like(q, 7)
    call(gb, kernels, B, q, 8, 0.125, out)
    torch.cuda.synchronize()
    assert out[:n].isnan().all() and (out[n] == 0).all() and out[n + 1:].isfinite().all()


@pytest.mark.parametrize("typ", TYPES)
def test_scores_of_minus_infinity_beside_others(gb, kernels, cuda, typ):
    # the first positions' scores are -infinity: the rows that see no others are NaN, later rows leave them out
    n = 300
    B = Batch([(n, n)], 2, 64, 16, typ, 330)
    q = queries(B, 8)
    place(B, 0, 0, 5, k=-1000.0)
    out = torch.zeros_like(q)
    want, mag, _ = B.attention(q, 8, 0.125, out)  # of a score of -8000: a weight of zero
    place(B, 0, 0, 5, k=-math.inf)
    call(gb, kernels, B, q, 8, 0.125, out)
    torch.cuda.synchronize()
    pages, slot = B.slots(0, 5, n)
    big = float(B.k[pages, :, slot].double().abs().sum(-1).max()) * 0.125
    assert out[:5].isnan().all()
    assert ((out.double() - want).abs() <= bound(typ, 64, n, want, mag, big))[5:].all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("rows", [1, 25, 39])
def test_a_call_of_the_first_rows(gb, kernels, cuda, typ, rows):
    # the call's rows end within a sequence's: those it has stand where they stand in the whole, as in the append
    B = Batch([(3, 70), (37, 400)], 2, 64, 16, typ, 340)
    q = torch.randn((B.rows, 8 * 64), generator=torch.Generator().manual_seed(9)).to(DT[typ]).cuda()
    out = torch.full_like(q, 7)
    want, mag, big = B.attention(q, 8, 0.125, out)
    c = B.chunk(gb)
    c.rows = rows
    kernels.attn_chunk_paged(c, q, q.stride(0), 8, 0.125, out, out.stride(0))
    torch.cuda.synchronize()
    assert ((out.double() - want).abs() <= bound(typ, 64, 400, want, mag, big))[:rows].all()
    assert (out[rows:] == 7).all()


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("heads,n", [(1, 1), (4, 1), (4, 32), (128, 1)])
def test_few_rows_keep_their_weights(gb, kernels, cuda, typ, heads, n):
    # Up to 128 packed rows hold a weight in two parts of the type: what is left of it is the square of a half step,
    # nothing of the half step itself. Weights of 1 and 0.7519, which lies between the numbers of both types, on
    # values that leave little of their sum: the second rounded once (by 7.5e-5 of it in binary16, 2.5e-3 in
    # bfloat16) would be off by 2.5 times what is allowed here and more.
    kv = 128
    B = Batch([(n, kv)], 1, 64, 16, typ, 350)
    k = torch.zeros(kv, dtype=torch.float64)
    k[1::2] = -146 / 4096  # exact scores: 0 and -0.28515625
    v = torch.ones(kv, dtype=torch.float64)
    v[1::2] = -1.3330
    place(B, 0, 0, kv, k=k, v=v)
    q = queries(B, heads)
    out = torch.zeros_like(q)
    want, mag, big = B.attention(q, heads, 0.125, out)
    call(gb, kernels, B, q, heads, 0.125, out)
    torch.cuda.synchronize()
    u = half_step(typ)
    # no error of a score; of a weight the remainder's own half step
    tol = u * want.abs() + (u * u + 2.0 ** -20 + kv * 2.0 ** -23) * mag
    assert ((out.double() - want).abs() <= tol).all(), float((out.double() - want).abs().max())


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n,kv", [(256, 4096), (1, 4096)])
@pytest.mark.parametrize("where", ["one value", "all values", "one key"])
def test_a_nan_that_all_rows_see_costs_little(gb, kernels, cuda, typ, n, kv, where):
    # Rows are done again, each by itself, for what a row they share a tile with sees and they do not. A NaN that a
    # row sees is no reason: all of a prompt's rows done again took 1,900 times a call's time.
    B = Batch([(n, kv)] * (1 if n > 1 else 16), 8, 128, 16, typ, 360)
    q = torch.randn((B.rows, 32 * 128), generator=torch.Generator().manual_seed(10)).to(DT[typ]).cuda()
    out = torch.zeros_like(q)

    def took():
        best = 1e9
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call(gb, kernels, B, q, 32, 0.1, out)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best
    clean = took()
    assert out.isfinite().all()
    for b in range(B.batch):
        if where == "one value":
            place(B, b, 10, 11, v=math.nan)
        elif where == "all values":
            place(B, b, 0, kv, v=math.nan)
        else:
            place(B, b, 10, 11, k=math.nan)
    spoilt = took()
    assert out.isnan().all()
    assert spoilt < 20 * clean, (spoilt, clean)


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("n,kv", [(1, 300), (100, 300), (100, 3000)])
def test_an_infinite_value_shows_as_one(gb, kernels, cuda, typ, n, kv):
    # at one position and in one dimension, with a weight like the others': the rows that see it have it there, and
    # nothing else changes
    B = Batch([(n, kv), (2, 50)], 2, 64, 16, typ, 370)
    q = 0.1 * torch.randn((B.rows, 8 * 64), generator=torch.Generator().manual_seed(11))
    q, out = q.to(DT[typ]).cuda(), torch.zeros((B.rows, 8 * 64), dtype=DT[typ], device="cuda")
    want, mag, big = B.attention(q, 8, 0.125, out)
    at = kv - 1 - n // 2
    pages, slot = B.slots(0, at, at + 1)
    B.v[pages, :, slot, 5] = -math.inf
    call(gb, kernels, B, q, 8, 0.125, out)
    torch.cuda.synchronize()
    first = at - (kv - n)
    shows = out[first:n].reshape(n - first, 8, 64)[..., 5]
    assert (shows == -math.inf).all()
    out[first:n].reshape(n - first, 8, 64)[..., 5] = want[first:n].reshape(n - first, 8, 64)[..., 5].to(out.dtype)
    assert ((out.double() - want).abs() <= bound(typ, 64, kv, want, mag, big)).all()
