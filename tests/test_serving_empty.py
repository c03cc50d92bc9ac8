"""Steps without rows or sequences: an empty buffer's address may be null."""
import ctypes as C

import pytest


def chunk(gb, rows, batch):
    return gb.paged_chunk(rows, batch, None, None, None, 8, 32, 16, 2, 64, gb.F16, None, None)


def calls(gb, h, c, rows):
    lib, rope = gb.lib(), gb.rope(1e4, 64)
    return [lib.gb_gpu_attn_chunk_paged(h, None, C.byref(c), None, 512, 8, 0.125, None, 512),
            lib.gb_gpu_rope_append_paged(h, None, C.byref(c), gb.F16, None, 512, 8, None, 128, None, 128, None,
                                         C.byref(rope), None, 512)] + (
           [] if rows else [lib.gb_gpu_qk_norm_rope(h, None, gb.F16, None, 512, 8, None, 128, 2, 0, 64, None,
                                                    C.byref(rope), None, gb.F16, None, 512, None, 128)])


@pytest.mark.parametrize("rows,batch", [(0, 3), (5, 0), (0, 0)])
def test_only_the_handle_is_missed(gb, rows, batch):
    for rc in calls(gb, None, chunk(gb, rows, batch), rows):
        assert rc == 1 and "not loaded" in gb.lib().gb_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,batch", [(0, 3), (5, 0), (0, 0)])
def test_nothing_is_done(gb, kernels, cuda, rows, batch):
    assert set(calls(gb, kernels.h, chunk(gb, rows, batch), rows)) == {0}


def test_rows_need_their_buffers(gb):
    for rc in calls(gb, None, chunk(gb, 5, 3), 5):
        assert rc == 1 and "bad arguments" in gb.lib().gb_last_error().decode()
