"""Per-head norms and rotation over so many rows that a CTA takes four
(gb_gpu_qk_norm_rope): the last CTA with fewer, lanes past head_dim, several
slices of the heads, the sizes just below."""
import pytest
import torch

from serving_ref import DT, norm, rotate
from test_qk_rows_gpu import close, make, size_of

pytestmark = pytest.mark.gpu

FULL = 4 * 6 * 740  # rows of one slice from which four go to a CTA


@pytest.mark.parametrize("typ,out", [("f16", "f16"), ("bf16", "bf16"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("nq,nk,hd,rows", [(20, 4, 80, FULL - 2), (20, 4, 80, FULL - 4), (14, 2, 128, FULL + 1),
                                           (28, 4, 64, FULL), (64, 8, 112, FULL // 3 + 3), (24, 8, 16, FULL * 4 + 2)])
def test_four_rows_to_a_cta(gb, kernels, cuda, typ, out, nq, nk, hd, rows):
    g = torch.Generator().manual_seed(8)
    qk = make(rows, nq + nk, hd, typ, 211, 2.0)
    pos = torch.randint(0, 100000, (rows,), generator=g, dtype=torch.int32).cuda()
    w = (1 + 0.3 * torch.randn(hd, generator=g)).cuda()
    wide, e = (nq + nk) * hd, qk.element_size()
    got = torch.full((rows, wide + 8), 3.0, dtype=DT[out], device="cuda")
    at, to = qk.data_ptr(), got.data_ptr()
    for wq, wk in ((w, w), (None, w), (None, None)):
        nrm = gb.qk_norm(wq, wk, 1e-6) if wk is not None else None
        kernels.qk_norm_rope(getattr(gb, typ.upper()), at, wide, nq, at + nq * hd * e, wide, nk, rows, hd, nrm,
                             gb.rope(5e5, hd, True), pos, getattr(gb, out.upper()), to, wide + 8, to + nq * hd * e, wide + 8)
        torch.cuda.synchronize()
        x = qk.double().reshape(rows, nq + nk, hd)
        y = torch.cat((norm(x[:, :nq], wq, 1e-6), norm(x[:, nq:], wk, 1e-6)), 1)
        close(got[:, :wide].reshape(rows, nq + nk, hd), rotate(y, pos, hd, True, 5e5), size_of(y, hd, True), out)
        assert (got[:, wide:] == 3).all()
