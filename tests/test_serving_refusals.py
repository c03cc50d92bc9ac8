"""What the serving-step entry points refuse, by status and message, and the
arithmetic that cuts a batch's attention among CTAs: both without a GPU (the
arguments are checked before the handle, which is not given here)."""
import ctypes as C

import pytest


def chunk(gb, **kw):
    a = dict(rows=4, batch=2, q_start=4096, kv_lens=4096, block_table=4096, max_pages=8, n_pages=32, page_size=16,
             n_kv=2, head_dim=64, kv_typ=gb.F16, k_pool=4096, v_pool=4096)
    a.update(kw)
    return gb.paged_chunk(**a)


def refused(gb, rc, code, word):
    msg = gb.lib().gb_last_error().decode()
    assert rc == code and word in msg, (rc, msg)


def attn(gb, c, q=4096, ldq=512, heads=8, scale=0.125, out=4096, ldo=512):
    return gb.lib().gb_gpu_attn_chunk_paged(None, None, C.byref(c) if c else None, q, ldq, heads, scale, out, ldo)


@pytest.mark.parametrize("what,code,word", [
    (dict(rows=-1), 1, "bad arguments"), (dict(batch=-1), 1, "bad arguments"), (dict(max_pages=0), 1, "bad arguments"),
    (dict(n_pages=0), 1, "bad arguments"), (dict(page_size=0), 1, "bad arguments"), (dict(n_kv=0), 1, "bad arguments"),
    (dict(q_start=None), 1, "bad arguments"), (dict(kv_lens=None), 1, "bad arguments"),
    (dict(block_table=None), 1, "bad arguments"), (dict(k_pool=None), 1, "pools"), (dict(v_pool=4104), 1, "pools"),
    (dict(max_pages=1 << 28, page_size=1 << 4), 1, "positions"), (dict(kv_typ=8), 3, "pool type 8"),
])
def test_chunk_description(gb, what, code, word):
    c = chunk(gb, **what)
    refused(gb, attn(gb, c), code, word)
    rc = gb.lib().gb_gpu_rope_append_paged(None, None, C.byref(c), gb.F16, 4096, 512, 8, 4096, 128, 4096, 128, None,
                                           None, 4096, 512)
    refused(gb, rc, code, word)


@pytest.mark.parametrize("what,more,code,word", [
    ({}, dict(heads=7), 1, "multiple of 2 KV heads"), ({}, dict(heads=0), 1, "KV heads"), ({}, dict(q=None), 1, "null"),
    ({}, dict(out=None), 1, "null"), ({}, dict(q=4100), 1, "16-byte"), ({}, dict(scale=0.0), 1, "scale"),
    ({}, dict(scale=float("nan")), 1, "scale"), ({}, dict(scale=float("inf")), 1, "scale"),
    ({}, dict(ldq=508), 1, "apart"), ({}, dict(ldo=504), 1, "apart"), (dict(head_dim=136), {}, 3, "head_dim 136"),
    (dict(head_dim=40), {}, 3, "head_dim 40"), (dict(head_dim=0), {}, 3, "head_dim 0"),
    (dict(rows=1 << 30), {}, 3, "rows of 8 heads"),
])
def test_attention(gb, what, more, code, word):
    refused(gb, attn(gb, chunk(gb, **what), **more), code, word)


def test_good_arguments_need_the_handle(gb):
    refused(gb, attn(gb, None), 1, "no chunk")
    refused(gb, attn(gb, chunk(gb)), 1, "not loaded")
    c = chunk(gb)
    rc = gb.lib().gb_gpu_rope_append_paged(None, None, C.byref(c), gb.F32, None, 0, 0, 4096, 128, 4096, 128, None, None,
                                           None, 0)
    refused(gb, rc, 1, "not loaded")
    refused(gb, norm(gb), 1, "not loaded")


def norm(gb, typ=0, q=4096, ldq=512, heads=8, k=4096, ldk=128, kv=2, rows=4, hd=64, nrm=None, rope=None, pos=4096,
         out=1, q_out=4096, ldqo=512, k_out=4096, ldko=128):
    return gb.lib().gb_gpu_qk_norm_rope(None, None, typ, q, ldq, heads, k, ldk, kv, rows, hd,
                                        C.byref(nrm) if nrm else None, C.byref(rope) if rope else None, pos, out, q_out,
                                        ldqo, k_out, ldko)


def test_norm_and_rotation(gb):
    r = gb.rope
    for more, code, word in (
            (dict(typ=2), 3, "types 2"), (dict(out=14), 3, "types"), (dict(rows=-1), 1, "-1 rows"),
            (dict(rows=(1 << 30) + 1), 3, "rows"),
            (dict(heads=-1), 1, "query heads"), (dict(hd=24), 3, "head_dim 24"), (dict(hd=272), 3, "head_dim 272"),
            (dict(q=None), 1, "q is null"), (dict(q_out=None), 1, "q_out is null"), (dict(k=None), 1, "k is null"),
            (dict(k_out=4104), 1, "16-byte"), (dict(ldq=500), 1, "apart"), (dict(ldk=120), 1, "apart"),
            (dict(rope=r(1e4, 64), pos=None), 1, "pos is null"), (dict(rope=r(1e4, 72)), 3, "72 rotated dims"),
            (dict(rope=r(1e4, 80)), 3, "80 rotated dims"), (dict(rope=r(1e4, -16)), 3, "rotated dims"),
            (dict(rope=r(0.0, 64)), 1, "base"), (dict(rope=r(float("nan"), 64)), 1, "base"),
            (dict(rope=r(float("inf"), 64)), 1, "base"), (dict(nrm=gb.qk_norm(4096, 4100, 1e-5)), 1, "weights"),
            (dict(nrm=gb.qk_norm(4096, 4096, -1.0)), 1, "eps"), (dict(nrm=gb.qk_norm(4096, 4096, float("nan"))), 1, "eps")):
        refused(gb, norm(gb, **more), code, word)


# ---- the line of work (gb_chunk.cu), restated ---------------------------------


def line_pieces(seqs, G, n_kv, RU, KT, grid, wide, narrow, opening, cap=1 << 30):
    """Every CTA's pieces (CTA, sequence, unit, head, t0, t1, tiles, c_first, c_last) as the kernel walks them."""
    def tiles(n, kv, u):
        last = min(n * G, (u + 1) * RU) - 1
        vis = max(0, min(min(max(kv, 0), cap), max(kv, 0) - n + last // G + 1))
        return max(1, -(-vis // KT))

    def cost(n, u):
        return wide if n * G - u * RU > RU // 2 else narrow
    units = [-(-n * G // RU) for n, _ in seqs]
    line = [(b, u, h) for b in range(len(seqs)) for u in range(units[b]) for h in range(n_kv)]
    begin, total = {}, 0
    for b, u, h in line:
        begin[b, u, h] = total
        total += opening + tiles(*seqs[b], u) * cost(seqs[b][0], u)
    many = len(seqs) <= 64 and all(n * G <= RU // 2 for n, _ in seqs)
    most = (narrow if many else wide) + opening
    ctas = min(grid, -(-total // most))
    while ctas > 1 and total < ctas * most:
        ctas -= 1
    got = []
    for me in range(grid):
        m = min(me, ctas)
        x0 = total * m // ctas if ctas else 0
        x1 = total * (m + 1) // ctas if m < ctas else x0
        for b, u, h in line:
            y, nt, c = begin[b, u, h], tiles(*seqs[b], u), cost(seqs[b][0], u)
            if y >= x1 or y + opening + nt * c <= x0:
                continue

            def tile_at(pos):
                return 0 if pos <= 0 else 1 if pos <= opening else -(-(pos - opening) // c)
            t0, t1 = tile_at(x0 - y), min(nt, tile_at(x1 - y))
            if t0 < t1:
                last = y + (opening + (nt - 1) * c if nt > 1 else 0)
                got.append((me, b, u, h, t0, t1, nt, ((y + 1) * ctas - 1) // total, ((last + 1) * ctas - 1) // total))
    return got, units, tiles


@pytest.mark.parametrize("RU,KT,grid,costs", [(64, 64, 296, (1, 1, 0)), (256, 128, 148, (4, 2, 2)), (64, 64, 3, (1, 1, 0)),
                                              (256, 128, 7, (4, 2, 2)), (256, 128, 148, (4, 2, 6)),
                                              (128, 64, 296, (1, 1, 0)), (64, 32, 296, (1, 1, 0))])
def test_every_tile_has_one_cta_and_every_unit_its_joiners(RU, KT, grid, costs):
    import random
    r = random.Random(RU + grid)
    for _ in range(40):
        seqs = [(r.choice([0, 1, 1, r.randint(1, 300)]), r.choice([0, r.randint(1, 40), r.randint(1, 6000)]))
                for _ in range(r.choice([1, 2, 9, 70]))]
        G, n_kv = r.choice([1, 3, 4, 8, 71]), r.choice([1, 2, 8])
        got, units, tiles = line_pieces(seqs, G, n_kv, RU, KT, grid, *costs)
        by = {}
        slots = set()
        for me, b, u, h, t0, t1, nt, first, last in got:
            assert 0 <= t0 < t1 <= nt == tiles(*seqs[b], u) and first <= me <= last < grid
            by.setdefault((b, u, h), []).append((me, t0, t1, nt, first, last))
            if not (t0 == 0 and t1 == nt):  # a partial: its slot is used once
                assert (me, t0 == 0) not in slots
                slots.add((me, t0 == 0))
        assert set(by) == {(b, u, h) for b in range(len(seqs)) for u in range(units[b]) for h in range(n_kv)}
        counters = set()
        for pieces in by.values():
            pieces.sort(key=lambda p: p[1])
            assert pieces[0][1] == 0 and pieces[-1][2] == pieces[0][3]
            assert all(a[2] == b[1] for a, b in zip(pieces, pieces[1:]))
            first, last = pieces[0][4], pieces[0][5]
            assert [p[0] for p in pieces] == list(range(first, last + 1))  # all of them arrive, none else
            if len(pieces) > 1:
                assert first not in counters  # one unit to a counter
                counters.add(first)
