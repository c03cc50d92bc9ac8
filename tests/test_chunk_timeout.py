"""Waits of the chunk attention that run out (gb_gpu_attn_chunk_wait_limit):
the call ends, the handle tells once (gb_gpu_attn_chunk_status), for replays of
captured launches too, and what it runs next is as ever."""
import pytest
import torch

from serving_ref import DT, Batch
from test_chunk_attention_gpu import call


def test_refusals(gb):
    lib = gb.lib()
    for call_, code, word in ((lambda: lib.gb_gpu_attn_chunk_status(None), 1, "not loaded"),
                           (lambda: lib.gb_gpu_attn_chunk_wait_limit(None, 5), 1, "not loaded"),
                           (lambda: lib.gb_gpu_attn_chunk_wait_limit(None, (1 << 20) + 1), 1, "polls")):
        assert call_() == code and word in lib.gb_last_error().decode()


@pytest.fixture
def own(gb, cuda):
    k = gb.Kernels(0)
    yield k
    k.close()


def ran_out(gb, k):
    torch.cuda.synchronize()
    try:
        k.attn_chunk_status()
    except gb.GollamaError as e:
        assert "ran out" in str(e)
        k.attn_chunk_status()  # told once
        return True
    return False


BATCHES = [  # heads, KV heads, head_dim, page size (7: no TMA), sequences
    (8, 2, 64, 16, [(1, 300), (40, 130), (2, 0), (70, 70)]),
    (8, 2, 128, 16, [(1, 9000), (100, 3000), (0, 50)]),
    (3, 1, 128, 24, [(200, 2000), (1, 128)]),
    (8, 2, 64, 7, [(1, 3000), (90, 500)]),
]


def batch(bi, typ):
    heads, n_kv, hd, page, seqs = BATCHES[bi]
    B = Batch(seqs, n_kv, hd, page, typ, 400, first=1, pad=2)
    q = torch.randn((B.rows, heads * hd), generator=torch.Generator().manual_seed(401)).to(DT[typ]).cuda()
    return B, q, heads


@pytest.mark.gpu
@pytest.mark.parametrize("typ", ["f16", "bf16"])
@pytest.mark.parametrize("bi", range(len(BATCHES)))
@pytest.mark.parametrize("polls", [0, 1, 3, 10, 30, 100, 1000])
def test_waits_that_run_out(gb, own, bi, typ, polls):
    B, q, heads = batch(bi, typ)
    out = torch.full_like(q, 7)
    call(gb, own, B, q, heads, 0.1, out)
    assert not ran_out(gb, own)
    want = out.clone()
    for _ in range(3):
        own.attn_chunk_wait_limit(polls)
        out.fill_(7)
        call(gb, own, B, q, heads, 0.1, out)
        late = ran_out(gb, own)
        assert late or polls
        assert late or torch.equal(out, want)
        assert (out[0] == 7).all() and (out[-2:] == 7).all()  # rows of no sequence, even so
        own.attn_chunk_wait_limit()
        call(gb, own, B, q, heads, 0.1, out)  # the workspace is as a call that ended leaves it
        assert not ran_out(gb, own) and torch.equal(out, want)


@pytest.mark.gpu
def test_the_next_call_tells(gb, own):
    B, q, heads = batch(0, "f16")
    out = torch.zeros_like(q)
    own.attn_chunk_wait_limit(0)
    call(gb, own, B, q, heads, 0.1, out)
    torch.cuda.synchronize()
    own.attn_chunk_wait_limit()
    out.fill_(7)
    with pytest.raises(gb.GollamaError, match="ran out"):
        call(gb, own, B, q, heads, 0.1, out)
    torch.cuda.synchronize()
    assert (out == 7).all()
    call(gb, own, B, q, heads, 0.1, out)
    assert not ran_out(gb, own) and out.isfinite().all() and not (out[1:-2] == 7).all()


@pytest.mark.gpu
def test_a_replay_tells(gb, own):
    B, q, heads = batch(1, "bf16")
    out = torch.zeros_like(q)
    call(gb, own, B, q, heads, 0.1, out)
    assert not ran_out(gb, own)
    want = out.clone()
    graphs = []
    for polls in (0, -1):
        own.attn_chunk_wait_limit(polls)
        graphs.append(torch.cuda.CUDAGraph())
        side = torch.cuda.Stream()
        with torch.cuda.graph(graphs[-1], stream=side):
            call(gb, own, B, q, heads, 0.1, out, stream=side)
    for _ in range(2):
        graphs[0].replay()
        assert ran_out(gb, own)
        out.zero_()
        graphs[1].replay()
        assert not ran_out(gb, own) and torch.equal(out, want)


@pytest.mark.gpu
def test_float32_waits_for_nothing(gb, own):
    B, q, heads = batch(0, "f32")
    out, again = torch.zeros_like(q), torch.zeros_like(q)
    call(gb, own, B, q, heads, 0.1, out)
    own.attn_chunk_wait_limit(0)
    call(gb, own, B, q, heads, 0.1, again)
    assert not ran_out(gb, own) and torch.equal(out, again)
