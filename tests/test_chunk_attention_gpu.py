"""Attention of new rows over the pages (gb_gpu_attn_chunk_paged) against the
plain 64-bit form: head layouts, ragged and empty batches, page sizes, lengths
from none to long, what lies in unused slots, streams, graphs and devices."""
import math

import pytest
import torch

from serving_ref import DT, Batch, half_step

pytestmark = pytest.mark.gpu


def bound(typ, hd, longest, want, mag, big):
    """Of each output: the rounding of the result, the rounding of the weights
    to the type (none in float32), twice the error of a score (hd products
    summed in float32, at worst truncated: hd 2^-23 of the sum of |q||k|), the
    exponential (2^-20), and a float32 sum over the positions (2^-23 each)."""
    u = half_step(typ)
    weights = 0.0 if typ == "f32" else 2 * u
    return u * want.abs() + (weights + 2 * hd * 2.0 ** -23 * big + 2.0 ** -20 + longest * 2.0 ** -23) * mag + 1e-30


def call(gb, kernels, B, q, n_heads, scale, out, stream=None):
    kernels.attn_chunk_paged(B.chunk(gb), q, q.stride(0), n_heads, scale, out, out.stride(0), stream=stream)


def run(gb, kernels, seqs, n_heads, n_kv, hd, page, typ, seed, spoil=False, ld_more=0, **kw):
    B = Batch(seqs, n_kv, hd, page, typ, seed, **kw)
    if spoil:  # unused slots and pages hold NaN and infinities
        used = torch.zeros((B.n_pages, page), dtype=torch.bool, device="cuda")
        for b, (_, kv) in enumerate(seqs):
            pages, slot = B.slots(b, 0, max(kv, 0))
            used[pages, slot] = True
        B.k.permute(0, 2, 1, 3)[~used] = float("nan")
        B.v.permute(0, 2, 1, 3)[~used] = float("inf")
    g = torch.Generator().manual_seed(seed + 1)
    wide = n_heads * hd
    q = (1.5 * torch.randn((B.rows, wide + ld_more), generator=g)).to(DT[typ]).cuda()
    out = torch.full((B.rows, wide + 2 * ld_more), 7.0, dtype=DT[typ], device="cuda")
    scale = 1 / math.sqrt(hd)
    want, mag, big = B.attention(q[:, :wide], n_heads, scale, out[:, :wide])
    for _ in range(2):  # the second call finds the workspace as the first left it
        out.fill_(7.0)
        call(gb, kernels, B, q, n_heads, scale, out)
        torch.cuda.synchronize()
        got = out[:, :wide].double()
        tol = bound(typ, hd, max([kv for _, kv in seqs] + [1]), want, mag, big)
        bad = ~((got - want).abs() <= tol)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got - want).abs().nan_to_num(9e9).max()))
        assert (out[:, wide:] == 7).all()
    return B, q, out


CASES = [  # heads, KV heads, head_dim, page size, (new rows, positions with them) of each sequence
    (8, 2, 64, 16, [(1, 1)]),
    (8, 2, 64, 16, [(1, 17), (5, 5), (3, 100), (1, 64)]),
    (32, 8, 128, 64, [(1, 300), (1, 1), (129, 1000), (64, 64), (2, 2)]),
    (32, 8, 128, 16, [(1, 8192)]),
    (32, 8, 128, 16, [(70, 2113)]),
    (6, 2, 96, 24, [(33, 4100), (1, 4099)]),
    (5, 1, 80, 7, [(50, 77), (1, 1000), (200, 201)]),
    (71, 1, 64, 32, [(9, 700), (1, 31)]),
    (4, 4, 16, 1, [(130, 130), (1, 259)]),
    (3, 3, 112, 256, [(257, 513), (128, 128), (127, 383)]),
    (64, 8, 128, 128, [(300, 2049)]),
    (16, 16, 128, 16, [(257, 257), (1, 4097)]),
]


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ci", range(len(CASES)))
def test_chunk_attention(gb, kernels, cuda, ci, typ):
    nh, nkv, hd, page, seqs = CASES[ci]
    run(gb, kernels, seqs, nh, nkv, hd, page, typ, 10 + ci)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_sequences_without_rows_or_positions(gb, kernels, cuda, typ):
    # no new rows; no positions; more new rows than positions (the first see nothing); rows of no sequence
    seqs = [(0, 40), (2, 0), (5, 2), (0, 0), (1, 9), (3, 3), (0, 7)]
    run(gb, kernels, seqs, 8, 2, 64, 16, typ, 40, first=3, pad=4)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_unused_slots_do_not_count(gb, kernels, cuda, typ):
    run(gb, kernels, [(1, 37), (40, 130), (2, 0), (1, 1)], 8, 2, 128, 16, typ, 50, spoil=True, pad=1)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_later_rows_do_not_reach_earlier_ones(gb, kernels, cuda, typ, value):
    # one position of the chunk holds NaN or an infinity in K and V: rows before it are as without it, and a NaN
    # shows in the rows from it on
    n, kv, at = 90, 700, 650
    B, q, clean = run(gb, kernels, [(n, kv), (1, 50)], 8, 2, 128, 16, typ, 60)
    clean = clean.clone()
    want, mag, big = B.attention(q, 8, 1 / math.sqrt(128), clean)
    pages, slot = B.slots(0, at, at + 1)
    B.k[pages, :, slot] = value
    B.v[pages, :, slot] = value
    out = torch.zeros_like(clean)
    call(gb, kernels, B, q, 8, 1 / math.sqrt(128), out)
    torch.cuda.synchronize()
    before = at - (kv - n)
    # such rows are summed in another order than the clean ones: a float32 sum over 700 positions may differ by
    # 700 2^-23 = 8.3e-5 of sum p |v| between orders, so each is held to the 64-bit form within its bound
    tol = bound(typ, 128, kv, want, mag, big)
    assert ((out[:before].double() - want[:before]).abs() <= tol[:before]).all()
    assert torch.equal(out[n:], clean[n:])
    if math.isnan(value):
        assert out[before:n].isnan().all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_more_sequences_than_threads(gb, kernels, cuda, typ):
    seqs = [(1 + (b * 7) % 3, 3 + (b * 37) % 190) for b in range(1100)]
    seqs[500] = (0, 5)
    run(gb, kernels, seqs, 4, 1, 64, 16, typ, 70)


@pytest.mark.parametrize("typ", ["f32", "f16"])
def test_rows_apart(gb, kernels, cuda, typ):
    run(gb, kernels, [(5, 50), (1, 3)], 4, 2, 48, 16, typ, 80, ld_more=24)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_extreme_scores(gb, kernels, cuda, typ):
    # one key outweighs all others by more than the type's range; all scores alike; scores far below zero
    B = Batch([(40, 300)], 2, 64, 16, typ, 90)
    q = torch.randn((B.rows, 8 * 64), generator=torch.Generator().manual_seed(1)).to(DT[typ]).cuda()
    for how in ("peak", "flat", "low"):
        pages, slot = B.slots(0, 0, 300)
        if how == "peak":
            q = q * 0 + 8
            p, s = B.slots(0, 200, 201)
            B.k[p, :, s] = 30
        elif how == "flat":
            B.k.zero_()
        else:
            B.k.fill_(-30)
        out = torch.zeros_like(q)
        want, mag, big = B.attention(q, 8, 0.125, out)
        call(gb, kernels, B, q, 8, 0.125, out)
        torch.cuda.synchronize()
        assert ((out.double() - want).abs() <= bound(typ, 64, 300, want, mag, min(big, 100.0))).all(), how


def test_scores_grow_along_the_positions(gb, kernels, cuda):
    # every tile raises the running maximum: each earlier sum is scaled down again
    for typ in ("f32", "f16", "bf16"):
        B = Batch([(3, 1500)], 1, 64, 16, typ, 95)
        pages, slot = B.slots(0, 0, 1500)
        B.k[pages, :, slot] = (torch.arange(1500, device="cuda")[:, None, None] / 64).to(DT[typ])
        q = torch.ones((3, 4 * 64), dtype=DT[typ], device="cuda")
        out = torch.zeros_like(q)
        want, mag, big = B.attention(q, 4, 0.125, out)
        call(gb, kernels, B, q, 4, 0.125, out)
        torch.cuda.synchronize()
        # the scores are exact here (sums of multiples of 2^-8 below 2^11): no error of a score
        assert ((out.double() - want).abs() <= bound(typ, 64, 1500, want, mag, 1.0)).all(), typ


def test_table_entries_outside_the_pool_read_page_0(gb, kernels, cuda):
    B = Batch([(2, 40)], 2, 64, 16, "f16", 100)
    q = torch.randn((2, 4 * 64), generator=torch.Generator().manual_seed(2)).half().cuda()
    B.table[0, 1] = 0
    out, out2 = torch.zeros_like(q), torch.ones_like(q)
    call(gb, kernels, B, q, 4, 0.125, out)
    for bad in (-5, B.n_pages, 1 << 30):
        B.table[0, 1] = bad
        call(gb, kernels, B, q, 4, 0.125, out2)
        torch.cuda.synchronize()
        assert torch.equal(out, out2)


def test_lengths_past_the_table_and_rows_past_the_call(gb, kernels, cuda):
    # what the device arrays say is held to the buffers: kv_lens above the table's positions count as these, rows
    # past the call's do not exist, and a q_start that falls has no rows
    B = Batch([(2, 48)], 2, 64, 16, "f16", 101, wide_table=0)
    q = torch.randn((2, 4 * 64), generator=torch.Generator().manual_seed(3)).half().cuda()
    full, out = torch.zeros_like(q), torch.zeros_like(q)
    B.kv_lens.fill_(50)  # rows at positions 48 and 49 of a table of 48: both see all of it
    call(gb, kernels, B, q, 4, 0.125, full)
    B.kv_lens.fill_(2000000000)
    call(gb, kernels, B, q, 4, 0.125, out)
    torch.cuda.synchronize()
    assert torch.equal(out, full)
    B.kv_lens.fill_(48)
    B.q_start.copy_(torch.tensor([0, 1 << 30], dtype=torch.int32))
    call(gb, kernels, B, q, 4, 0.125, out)
    B.q_start.copy_(torch.tensor([2, 0], dtype=torch.int32))
    out.fill_(5)
    call(gb, kernels, B, q, 4, 0.125, out)
    torch.cuda.synchronize()
    assert (out == 5).all()


def test_streams_graphs_and_first_call(gb, cuda):
    k = gb.Kernels(0)
    try:
        B = Batch([(1, 900), (40, 333)], 2, 64, 16, "bf16", 110)
        q = torch.randn((B.rows, 8 * 64), generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
        out = torch.zeros_like(q)
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        # the first call allocates: refused inside a capture, which goes on
        with torch.cuda.graph(graph, stream=side):
            out.zero_()
            with pytest.raises(gb.GollamaError):
                call(gb, k, B, q, 8, 0.125, out, stream=side)
        call(gb, k, B, q, 8, 0.125, out, stream=side)
        side.synchronize()
        want = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call(gb, k, B, q, 8, 0.125, out, stream=side)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        # the device arrays may change between replays: lengths and tables are read when it runs
        B.kv_lens[0] = 5
        want, mag, big = Batch.attention(_with(B, [(1, 5), (40, 333)]), q, 8, 0.125, out)
        graph.replay()
        torch.cuda.synchronize()
        assert ((out.double() - want).abs() <= bound("bf16", 64, 900, want, mag, big)).all()
    finally:
        k.close()


def _with(B, seqs):
    B.seqs = seqs
    return B


def test_result_is_the_same_every_time(gb, kernels, cuda):
    B = Batch([(37, 5000), (1, 3000)], 2, 128, 16, "f16", 120)
    q = torch.randn((B.rows, 8 * 128), generator=torch.Generator().manual_seed(5)).half().cuda()
    outs = []
    for _ in range(20):
        out = torch.zeros_like(q)
        call(gb, kernels, B, q, 8, 0.09, out)
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs)


def test_long_cache_offsets(gb, kernels, cuda):
    # a pool of more than 2^32 elements, the sequence's pages at its end
    page, hd, nkv = 64, 128, 8
    n_pages = (1 << 32) // (page * hd * nkv) + 40
    pool = torch.zeros((2, n_pages, nkv, page, hd), dtype=torch.float16, device="cuda")
    B = Batch([(3, 700)], nkv, hd, page, "f16", 130)
    far = n_pages - B.n_pages
    pool[0, far:], pool[1, far:] = B.k, B.v
    q = torch.randn((3, 32 * hd), generator=torch.Generator().manual_seed(6)).half().cuda()
    a, b = torch.zeros_like(q), torch.ones_like(q)
    call(gb, kernels, B, q, 32, 0.09, a)
    B.table[B.table >= 0] += far
    B.n_pages, B.k, B.v = n_pages, pool[0], pool[1]
    call(gb, kernels, B, q, 32, 0.09, b)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_two_handles_on_two_streams(gb, cuda):
    # a handle for each stream: calls that overlap on the GPU do not share a workspace
    batches = [Batch([(1, 3000), (1, 77)], 2, 64, 16, "f16", 140), Batch([(200, 900)], 2, 64, 16, "f16", 141)]
    ks, outs, wants = [gb.Kernels(0), gb.Kernels(0)], [], []
    try:
        qs = [torch.randn((B.rows, 8 * 64), generator=torch.Generator().manual_seed(i)).half().cuda()
              for i, B in enumerate(batches)]
        for B, q, k in zip(batches, qs, ks):
            out = torch.zeros_like(q)
            call(gb, k, B, q, 8, 0.125, out)
            torch.cuda.synchronize()
            wants.append(out.clone())
            outs.append(out.zero_())
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        for _ in range(20):
            for B, q, k, o, st in zip(batches, qs, ks, outs, streams):
                call(gb, k, B, q, 8, 0.125, o, stream=st)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
    finally:
        for k in ks:
            k.close()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,n", [(1, 127), (1, 128), (1, 129), (1, 255), (1, 256), (1, 257), (2, 64), (2, 65),
                                     (16, 1), (16, 8), (128, 1), (129, 1), (300, 1)])
def test_rows_around_a_units_borders(gb, kernels, cuda, typ, heads, n):
    # one KV head: `heads` packed rows for each new row, around 128 and 256 of them
    run(gb, kernels, [(n, n + 170), (n, n)], heads, 1, 32, 16, typ, 150)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page", [1, 8, 16, 24, 100, 128, 192])
def test_page_sizes_and_ends_within_a_tile(gb, kernels, cuda, typ, page):
    run(gb, kernels, [(1, 127), (1, 128), (1, 129), (3, 255), (3, 257), (1, 1), (40, 300)], 4, 2, 64, page, typ, 160,
        spoil=True)


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_nothing_to_do(gb, kernels, cuda, typ):
    B = Batch([(2, 20)], 2, 64, 16, typ, 170)
    q = torch.zeros((B.rows, 4 * 64), dtype=DT[typ], device="cuda")
    out = torch.full_like(q, 3)
    c = B.chunk(gb)
    for rows, batch in ((0, 1), (2, 0)):
        c.rows, c.batch = rows, batch
        kernels.attn_chunk_paged(c, q, 256, 4, 0.125, out, 256)
        kernels.rope_append_paged(c, getattr(gb, typ.upper()), None, 0, 0, q, 256, q, 256, None, None, 0)
    torch.cuda.synchronize()
    assert (out == 3).all()


@pytest.mark.parametrize("typ", ["f16", "bf16"])
def test_an_infinite_key_shows(gb, kernels, cuda, typ):
    # an infinite score makes the rows that see it NaN, as inf - inf does, and no other row
    B = Batch([(30, 400), (4, 90)], 2, 64, 16, typ, 180)
    q = torch.ones((B.rows, 4 * 64), dtype=DT[typ], device="cuda")
    pages, slot = B.slots(0, 10, 11)
    B.k[pages, :, slot] = float("inf")
    out = torch.zeros_like(q)
    call(gb, kernels, B, q, 4, 0.125, out)
    torch.cuda.synchronize()
    assert out[:30].isnan().all() and out[30:].isfinite().all()


def test_a_falling_q_start_has_no_rows(gb, kernels, cuda):
    # the difference of two of its entries may pass 32 bits
    B = Batch([(2, 48), (1, 9)], 2, 64, 16, "f16", 190)
    q = torch.randn((3, 4 * 64), generator=torch.Generator().manual_seed(7)).half().cuda()
    for starts in ([1, -2 ** 31, 0], [2 ** 31 - 1, -2 ** 31, -2 ** 31], [2 ** 31 - 1, 2 ** 31 - 1, 0]):
        B.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        out = torch.full_like(q, 5)
        call(gb, kernels, B, q, 4, 0.125, out)
        torch.cuda.synchronize()
        assert (out == 5).all(), starts


def test_a_unit_of_many_tiles(gb, cuda):
    # 2^22 positions, all of them the slots of one page: a unit of 256 rows takes 32768 tiles, and no wait that
    # spans them runs out (the next call would say so). Scores are zero and values one: sums of ones below 2^24
    # are exact, and their quotient is off by the reciprocal's and the product's half steps, which the result's
    # type rounds away.
    k = gb.Kernels(0)
    try:
        n, kv, page = 512, 1 << 22, 128
        pool = torch.zeros((2, 1, 1, page, 64), dtype=torch.float16, device="cuda")
        pool[1] = 1
        table = torch.zeros((1, kv // page), dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        lens = torch.tensor([kv], dtype=torch.int32, device="cuda")
        c = gb.paged_chunk(n, 1, starts, lens, table, kv // page, 1, page, 1, 64, gb.F16, pool[0], pool[1])
        heads = 148 * 256 // n  # enough rows for a whole unit or more to each CTA
        q = torch.ones((n, heads * 64), dtype=torch.float16, device="cuda")
        out = torch.zeros_like(q)
        for _ in range(2):
            k.attn_chunk_paged(c, q, heads * 64, heads, 0.125, out, heads * 64)
            torch.cuda.synchronize()
        assert (out == 1).all()
    finally:
        k.close()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,n", [(8, 9), (8, 40), (3, 30), (1, 140)])
def test_nan_queries_stay_in_their_rows(gb, kernels, cuda, typ, heads, n):
    # the rows behind a sequence's are another's (or nobody's), whatever they hold
    B = Batch([(n, 300), (7, 90), (n, n)], 1, 64, 16, typ, 200, pad=3)
    q = torch.randn((B.rows, heads * 64), generator=torch.Generator().manual_seed(8)).to(DT[typ]).cuda()
    out = torch.full_like(q, 7)
    want, mag, big = B.attention(q, heads, 0.125, out)
    q[n:n + 7], q[2 * n + 7:] = float("nan"), float("inf")
    call(gb, kernels, B, q, heads, 0.125, out)
    torch.cuda.synchronize()
    fine = ((out.double() - want).abs() <= bound(typ, 64, 300, want, mag, big)).all(1)
    assert fine[:n].all() and fine[n + 7:].all() and out[n:n + 7].isnan().all()
