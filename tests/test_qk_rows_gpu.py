"""Per-head norms with the rotation (gb_gpu_qk_norm_rope) and the paged append
(gb_gpu_rope_append_paged) against their plain 64-bit forms, and the serving
step they form with the chunk and decode attention."""
import math

import pytest
import torch

from serving_ref import DT, Batch, half_step, norm, rotate

pytestmark = pytest.mark.gpu

# Errors of the float32 arithmetic in units of 2^-24 of a pair's magnitude: the
# norm's sum (a tree of 8 levels over runs of 16), its root and two products
# (28 in all), the angle's rounding to float32 (pi 2^-24, as sine or cosine),
# sincospi (2 each), two products and a sum (3).
STEPS = 48


def close(got, want, size, typ):
    tol = half_step(typ) * want.abs() + STEPS * 2.0 ** -24 * size + 1e-38
    if typ == "f16":
        tol = tol + 2.0 ** -25  # half a step of the subnormal numbers
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double() - want).abs().max()))


def size_of(x, dims, halves):
    """Each element's pair magnitude |a| + |b|."""
    y = x.abs().clone()
    lo, hi = (slice(0, dims // 2), slice(dims // 2, dims)) if halves else (slice(0, dims, 2), slice(1, dims, 2))
    both = y[..., lo] + y[..., hi]
    y[..., lo], y[..., hi] = both, both
    return y


def make(rows, heads, hd, typ, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn((rows, heads * hd), generator=g)).to(DT[typ]).cuda()


NORM_CASES = [  # rows, query heads, KV heads, head_dim, rotated dims, halves, far
    (1, 32, 8, 128, 128, True, 8192),
    (1, 1, 0, 16, 16, False, 4),
    (7, 6, 2, 64, 64, False, 1 << 20),
    (61, 28, 4, 128, 64, False, 131072),
    (33, 71, 1, 80, 80, True, 1000),
    (5, 0, 3, 96, 48, True, 2047),
    (300, 64, 8, 256, 256, True, 131072),
    (19, 3, 3, 112, 16, False, 77),
    (4, 8, 8, 128, 0, False, 1),
]


@pytest.mark.parametrize("typ,out", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"),
                                     ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("ci", range(len(NORM_CASES)))
def test_norm_rope(gb, kernels, cuda, ci, typ, out):
    rows, nq, nk, hd, dims, halves, far = NORM_CASES[ci]
    g = torch.Generator().manual_seed(ci)
    qkv = make(rows, nq + 2 * nk, hd, typ, 200 + ci, 2.0)
    pos = torch.randint(0, far, (rows,), generator=g, dtype=torch.int32).cuda()
    pos[0] = far - 1
    wq, wk = (1 + 0.3 * torch.randn(hd, generator=g)).cuda(), (1 + 0.3 * torch.randn(hd, generator=g)).cuda()
    freq = (1 + torch.rand(dims // 2, generator=g)).cuda() if ci % 2 and dims else None
    base, eps = 500000.0, 1e-6
    q_out = torch.full((rows, nq * hd + 8), 3.0, dtype=DT[out], device="cuda")
    k_out = torch.full((rows, nk * hd + 8), 3.0, dtype=DT[out], device="cuda")
    at, wide, e = qkv.data_ptr(), (nq + 2 * nk) * hd, qkv.element_size()
    kernels.qk_norm_rope(getattr(gb, typ.upper()), at, wide, nq, at + nq * hd * e, wide, nk, rows, hd,
                         gb.qk_norm(wq, wk, eps), gb.rope(base, dims, halves, freq), pos, getattr(gb, out.upper()),
                         q_out, nq * hd + 8, k_out, nk * hd + 8)
    torch.cuda.synchronize()
    x = qkv.double().reshape(rows, nq + 2 * nk, hd)
    for got, xs, w, many in ((q_out, x[:, :nq], wq, nq), (k_out, x[:, nq:nq + nk], wk, nk)):
        y = norm(xs, w, eps)
        close(got[:, :many * hd].reshape(rows, many, hd), rotate(y, pos, dims, halves, base, freq),
              size_of(y, dims, halves), out)
        assert (got[:, many * hd:] == 3).all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nq,nk,hd,dims,halves,extra", [(5, 1, 80, 80, True, 0), (3, 2, 96, 32, False, 1),
                                                        (12, 2, 128, 128, True, 5), (1, 1, 48, 48, False, 2),
                                                        (40, 4, 256, 128, True, 3)])
def test_many_rows(gb, kernels, cuda, typ, nq, nk, hd, dims, halves, extra):
    # several rows to a CTA (from 2^26 elements on), the last of them with fewer; head_dims that leave lanes over
    rows = -(-(1 << 26) // (4 * (nq + nk) * hd)) * 4 + extra
    g = torch.Generator().manual_seed(7)
    qk = make(rows, nq + nk, hd, typ, 210, 2.0)
    pos = torch.randint(0, 100000, (rows,), generator=g, dtype=torch.int32).cuda()
    w = (1 + 0.3 * torch.randn(hd, generator=g)).cuda()
    q_out, k_out = torch.zeros((rows, nq * hd), dtype=DT[typ], device="cuda"), torch.zeros((rows, nk * hd), dtype=DT[typ], device="cuda")
    T, at, wide = getattr(gb, typ.upper()), qk.data_ptr(), (nq + nk) * hd
    kernels.qk_norm_rope(T, at, wide, nq, at + nq * hd * qk.element_size(), wide, nk, rows, hd, gb.qk_norm(w, w, 1e-6),
                         gb.rope(5e5, dims, halves), pos, T, q_out, nq * hd, k_out, nk * hd)
    torch.cuda.synchronize()
    y = norm(qk.double().reshape(rows, nq + nk, hd), w, 1e-6)
    want, size = rotate(y, pos, dims, halves, 5e5), size_of(y, dims, halves)
    close(q_out.reshape(rows, nq, hd), want[:, :nq], size[:, :nq], typ)
    close(k_out.reshape(rows, nk, hd), want[:, nq:], size[:, nq:], typ)
    # in place, and the same result
    kernels.qk_norm_rope(T, at, wide, nq, at + nq * hd * qk.element_size(), wide, nk, rows, hd, gb.qk_norm(w, w, 1e-6),
                         gb.rope(5e5, dims, halves), pos, T, at, wide, at + nq * hd * qk.element_size(), wide)
    torch.cuda.synchronize()
    assert torch.equal(qk, torch.cat((q_out, k_out), 1))


@pytest.mark.parametrize("typ,pool", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
def test_append_many_rows(gb, kernels, cuda, typ, pool):
    # more sequences than a warp looks at together, several rows to a CTA across their borders, norms on the way
    seqs = [(37 + b % 5, 60 + b % 90) for b in range(70)] + [(0, 12), (1, 1)]
    nq, nk, hd = 3, 2, 80
    B = Batch(seqs, nk, hd, 16, pool, 320, first=5, pad=7)
    qkv = make(B.rows, nq + 2 * nk, hd, typ, 420)
    q_out = torch.full((B.rows, nq * hd), 3.0, dtype=DT[pool], device="cuda")
    w = (1 + 0.3 * torch.randn(hd, generator=torch.Generator().manual_seed(5))).cuda()
    kp, vp, ksize = B.k.double().clone(), B.v.double().clone(), torch.zeros(B.k.shape, dtype=torch.float64, device="cuda")
    at, wide, e = qkv.data_ptr(), (nq + 2 * nk) * hd, qkv.element_size()
    kernels.rope_append_paged(B.chunk(gb), getattr(gb, typ.upper()), at, wide, nq, at + nq * hd * e, wide,
                              at + (nq + nk) * hd * e, wide, gb.rope(5e5, hd, True), q_out, nq * hd,
                              norm=gb.qk_norm(w, w, 1e-5))
    torch.cuda.synchronize()
    x = qkv.double().reshape(B.rows, nq + 2 * nk, hd)
    want, qsize = torch.full((B.rows, nq, hd), 3.0, dtype=torch.float64, device="cuda"), torch.zeros((B.rows, nq, hd), device="cuda")
    for b, (n, kv) in enumerate(seqs):
        r = slice(B.starts[b], B.starts[b] + n)
        y = norm(x[r, :nq + nk], w, 1e-5)
        z, size = rotate(y, torch.arange(kv - n, kv, device="cuda"), hd, True, 5e5), size_of(y, hd, True)
        want[r], qsize[r] = z[:, :nq], size[:, :nq]
        pages, slot = B.slots(b, kv - n, kv)
        kp[pages, :, slot], vp[pages, :, slot], ksize[pages, :, slot] = z[:, nq:], x[r, nq + nk:], size[:, nq:].double()
    close(q_out.reshape(B.rows, nq, hd), want, qsize, pool)
    close(B.k, kp, ksize, pool)
    assert torch.equal(B.v, vp.to(DT[pool]))


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("halves", [False, True])
def test_in_place_and_parts(gb, kernels, cuda, typ, halves):
    # norms alone, the rotation alone, a norm of the keys alone; each output in its input's place
    rows, nq, nk, hd = 9, 6, 2, 64
    pos = torch.arange(rows, dtype=torch.int32, device="cuda") * 17
    w = (1 + 0.1 * torch.arange(hd, device="cuda").float()) / 4
    T = getattr(gb, typ.upper())
    for nrm, rp in ((gb.qk_norm(w, w, 1e-5), None), (None, gb.rope(1e4, 64, halves)),
                    (gb.qk_norm(None, w, 1e-5), gb.rope(1e4, 32, halves))):
        q, k = make(rows, nq, hd, typ, 1), make(rows, nk, hd, typ, 2)
        q0, k0 = q.double().reshape(rows, nq, hd), k.double().reshape(rows, nk, hd)
        kernels.qk_norm_rope(T, q, nq * hd, nq, k, nk * hd, nk, rows, hd, nrm, rp, pos, T, q, nq * hd, k, nk * hd)
        torch.cuda.synchronize()
        dims = rp.dims if rp else 0
        for got, x, wt in ((q, q0, nrm and nrm.wq and w), (k, k0, nrm and nrm.wk and w)):
            y = norm(x, wt if torch.is_tensor(wt) else None, 1e-5)
            close(got.reshape(x.shape), rotate(y, pos, dims, halves, 1e4), size_of(y, dims, halves), typ)


def test_norm_of_zeros_and_infinities(gb, kernels, cuda):
    x = torch.zeros((3, 2 * 64), device="cuda")
    x[1, 5] = float("inf")
    x[2, 70] = float("nan")
    w = torch.ones(64, device="cuda")
    out = torch.ones_like(x)
    kernels.qk_norm_rope(gb.F32, x, 128, 2, None, 0, 0, 3, 64, gb.qk_norm(w, None, 1e-6), None, None, gb.F32, out, 128,
                         None, 0)
    torch.cuda.synchronize()
    assert (out[0] == 0).all() and out[1, 5].isnan() and (out[1, 64:] == 0).all()
    assert out[2, 64:].isnan().all() and (out[2, :64] == 0).all()


APPEND_CASES = [  # query heads, KV heads, head_dim, dims, halves, page size, (new rows, positions with them)
    (32, 8, 128, 128, False, 16, [(1, 4000), (1, 1), (1, 17)]),
    (6, 2, 64, 64, True, 24, [(50, 50), (3, 100), (0, 9), (100, 1000)]),
    (71, 1, 80, 32, True, 7, [(20, 33), (1, 1)]),
    (0, 4, 16, 16, False, 1, [(130, 130), (2, 70)]),
    (8, 8, 256, 256, True, 256, [(300, 700)]),
    (4, 4, 96, 0, False, 64, [(65, 129), (1, 2)]),
]


@pytest.mark.parametrize("typ,pool", [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("ci", range(len(APPEND_CASES)))
@pytest.mark.parametrize("normed", [False, True])
def test_append(gb, kernels, cuda, ci, typ, pool, normed):
    nq, nk, hd, dims, halves, page, seqs = APPEND_CASES[ci]
    B = Batch(seqs, nk, hd, page, pool, 300 + ci, first=2, pad=3)
    rows = B.rows
    qkv = make(rows, nq + 2 * nk, hd, typ, 400 + ci)
    q_out = torch.full((rows, nq * hd + 8), 3.0, dtype=DT[pool], device="cuda")
    w = (1 + 0.3 * torch.randn(hd, generator=torch.Generator().manual_seed(ci))).cuda() if normed else None
    nrm = gb.qk_norm(w, w, 1e-5) if normed else None
    kp, vp = B.k.double().clone(), B.v.double().clone()
    ksize = torch.zeros_like(kp)
    at, wide, e = qkv.data_ptr(), (nq + 2 * nk) * hd, qkv.element_size()
    kernels.rope_append_paged(B.chunk(gb), getattr(gb, typ.upper()), at if nq else None, wide, nq, at + nq * hd * e, wide,
                              at + (nq + nk) * hd * e, wide, gb.rope(5e5, dims, halves), q_out if nq else None,
                              nq * hd + 8, norm=nrm)
    torch.cuda.synchronize()
    x = qkv.double().reshape(rows, nq + 2 * nk, hd)
    want_q, qsize = torch.full((rows, nq, hd), 3.0, dtype=torch.float64, device="cuda"), torch.zeros((rows, nq, hd), device="cuda")
    for b, (n, kv) in enumerate(seqs):
        r = slice(B.starts[b], B.starts[b] + n)
        pos = torch.arange(kv - n, kv, device="cuda")
        y = norm(x[r, :nq + nk], w, 1e-5)
        z, size = rotate(y, pos, dims, halves, 5e5), size_of(y, dims, halves)
        want_q[r], qsize[r] = z[:, :nq], size[:, :nq]
        pages, slot = B.slots(b, kv - n, kv)
        kp[pages, :, slot], vp[pages, :, slot], ksize[pages, :, slot] = z[:, nq:], x[r, nq + nk:], size[:, nq:].double()
    close(q_out[:, :nq * hd].reshape(rows, nq, hd), want_q, qsize, pool)
    assert (q_out[:, nq * hd:] == 3).all()
    close(B.k, kp, ksize, pool)  # untouched slots: exactly as they were, up to the bound's 1e-38
    assert torch.equal(B.v, vp.to(DT[pool]))


def test_append_skips_bad_pages_and_positions(gb, kernels, cuda):
    B = Batch([(4, 40), (3, 1), (2, 9)], 2, 64, 16, "f16", 500, wide_table=0)
    B.table[0, 2] = B.n_pages + 5  # positions 36..39 of sequence 0 are on no page
    B.kv_lens[2] = 500             # past the table
    k0, v0 = B.k.clone(), B.v.clone()
    qkv = make(B.rows, 4 + 4, 64, "f16", 501)
    q_out = torch.zeros((B.rows, 4 * 64), dtype=torch.float16, device="cuda")
    at = qkv.data_ptr()
    kernels.rope_append_paged(B.chunk(gb), gb.F16, at, 512, 4, at + 512, 512, at + 768, 512, gb.rope(1e4, 64), q_out, 256)
    torch.cuda.synchronize()
    # sequence 1 has positions -2, -1, 0: the last alone is appended
    pages, slot = B.slots(1, 0, 1)
    assert torch.equal(B.v[pages, :, slot].flatten(), qkv[6, 384:])
    k1, v1 = B.k.clone(), B.v.clone()
    k1[pages, :, slot], v1[pages, :, slot] = k0[pages, :, slot], v0[pages, :, slot]
    assert torch.equal(k1, k0) and torch.equal(v1, v0)
    assert (q_out != 0).any(1).all()


@pytest.mark.parametrize("typ", ["f32", "f16", "bf16"])
def test_serving_step(gb, kernels, cuda, typ):
    """Norms and rotation, append and attention as a step runs them, on a stream of its own and captured, against
    the same in 64 bits; then a decode of each sequence through gb_gpu_attn_decode_paged."""
    nq, nk, hd, page = 8, 2, 64, 16
    seqs = [(1, 100), (45, 61), (7, 7), (1, 1)]
    B = Batch(seqs, nk, hd, page, typ, 600)
    qkv = make(B.rows, nq + 2 * nk, hd, "f32", 601)
    w = (1 + 0.1 * torch.randn(hd, generator=torch.Generator().manual_seed(3))).cuda()
    T, P = gb.F32, getattr(gb, typ.upper())
    at, wide = qkv.data_ptr(), (nq + 2 * nk) * hd
    q = torch.zeros((B.rows, nq * hd), dtype=DT[typ], device="cuda")
    out = torch.zeros_like(q)
    pos = torch.cat([torch.arange(kv - n, kv) for n, kv in seqs]).int().cuda()
    normed = torch.zeros((B.rows, (nq + nk) * hd), device="cuda")
    chunk, nrm, rp = B.chunk(gb), gb.qk_norm(w, w, 1e-5), gb.rope(1e4, hd, True)
    side = torch.cuda.Stream()
    args = (normed.data_ptr(), (nq + nk) * hd)

    def step():
        # as two calls (norm and rotation, then a plain append), as a program that needs the normed rows makes them
        kernels.qk_norm_rope(T, at, wide, nq, at + nq * hd * 4, wide, nk, B.rows, hd, nrm, rp, pos, T, *args,
                             normed.data_ptr() + nq * hd * 4, args[1], stream=side)
        kernels.rope_append_paged(chunk, T, *args, nq, normed.data_ptr() + nq * hd * 4, args[1],
                                  at + (nq + nk) * hd * 4, wide, None, q, nq * hd, stream=side)
        kernels.attn_chunk_paged(chunk, q, nq * hd, nq, 0.125, out, nq * hd, stream=side)

    torch.cuda.synchronize()
    step()
    side.synchronize()
    first, k1, v1, q1 = out.clone(), B.k.clone(), B.v.clone(), q.clone()
    x = qkv.double().reshape(B.rows, nq + 2 * nk, hd)
    z = rotate(norm(x[:, :nq + nk], w, 1e-5), pos, hd, True, 1e4)
    close(q.reshape(B.rows, nq, hd), z[:, :nq], 2 * z[:, :nq].abs().amax(-1, keepdim=True).expand_as(z[:, :nq]), typ)
    want, mag, big = B.attention(q, nq, 0.125, out)
    from test_chunk_attention_gpu import bound
    assert ((out.double() - want).abs() <= bound(typ, hd, 100, want, mag, big)).all()
    # one call with the norm inside gives the same cache and queries
    B.k.zero_(), B.v.zero_(), q.zero_()
    kernels.rope_append_paged(chunk, T, at, wide, nq, at + nq * hd * 4, wide, at + (nq + nk) * hd * 4, wide, rp, q,
                              nq * hd, norm=nrm, stream=side)
    side.synchronize()
    for b, (n, kv) in enumerate(seqs):
        pages, slot = B.slots(b, kv - n, kv)
        assert torch.equal(B.k[pages, :, slot], k1[pages, :, slot]) and torch.equal(B.v[pages, :, slot], v1[pages, :, slot])
    assert torch.equal(q, q1)
    # the step captured and replayed
    B.k.copy_(k1), B.v.copy_(v1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    if typ == "bf16":
        return
    # each sequence's last row once more by the decode attention (float32 queries)
    last = torch.tensor([B.starts[b + 1] - 1 for b in range(len(seqs))], device="cuda")
    q32, one = q[last].float().contiguous(), torch.zeros((len(seqs), nq * hd), device="cuda")
    kernels.attn_decode_paged(q32, B.k, B.v, typ == "f16", B.table, B.kv_lens, len(seqs), B.max_pages, B.n_pages, page,
                              nq, nk, hd, 0.125, one)
    torch.cuda.synchronize()
    tol = bound(typ, hd, 100, want, mag, big)[last] + 1e-5
    assert ((one.double() - out[last].double()).abs() <= 2 * tol).all()
