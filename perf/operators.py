"""The serving step's paged-cache operators as measured calls.

Three operators run one after another in a serving step whose K/V live in
pages of a shared pool [n_pages][n_kv][page_size][head_dim]:

``norm``    norms of queries and keys for each head, with the position
            rotation in the same pass
            x' = x / sqrt(mean(x^2) + eps) * w, then each pair (a, b) becomes
            (a cos t - b sin t, a sin t + b cos t), t = pos * base^(-2j/dims);
``append``  rotation of the new keys (and queries) and the append of keys and
            values at the sequences' next positions through their page tables;
``attn``    attention of each sequence's n new rows (1: decode) over its pages:
            row i of n attends to positions [0, kv_len - n + i].

A batch is described as the entry points take it: sequence b's new rows are
rows [q_start[b], q_start[b+1]) and kv_lens[b] counts its positions with them.
Where ``own`` is false ``run`` computes the plain forms in 32 bits (angles in
64); where it is true it calls the library.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -------------------------------------------------------------------


def listed():
    return [
        # one decoded token of the 8B shape: what a single user's step waits for
        {"name": "norm decode 1 row", "op": "norm", "rows": 1, "heads": 32, "kv": 8, "hd": 128, "dims": 128,
         "halves": True, "typ": "f32", "out": "f16", "far": 8192},
        # a batch of 61 sequences, pairs side by side as in the GGUF llama models, far positions
        {"name": "norm batch 61 rows", "op": "norm", "rows": 61, "heads": 28, "kv": 4, "hd": 128, "dims": 64,
         "halves": False, "typ": "bf16", "out": "bf16", "far": 131072},
        # the prompts of a full step of the 70B shape
        {"name": "norm prompt 8192 rows", "op": "norm", "rows": 8192, "heads": 64, "kv": 8, "hd": 128, "dims": 128,
         "halves": True, "typ": "f16", "out": "f16", "far": 16384},
        # 64 decoding sequences: one position each, float32 activations into a binary16 pool
        {"name": "append decode 64", "op": "append", "batch": 64, "new": 1, "ctx": 4096, "ragged": True, "pad": 0,
         "heads": 32, "kv": 8, "hd": 128, "dims": 128, "halves": False, "page": 16, "typ": "f32", "pool": "f16",
         "salt": 1},
        # a prompt chunk of one sequence, odd length and page size, rows of a padded batch behind it
        {"name": "append chunk 509", "op": "append", "batch": 1, "new": 509, "ctx": 2000, "ragged": False, "pad": 3,
         "heads": 32, "kv": 8, "hd": 64, "dims": 64, "halves": True, "page": 24, "typ": "bf16", "pool": "bf16",
         "salt": 2},
        # several prompts in one step
        {"name": "append prompts 8192", "op": "append", "batch": 7, "new": 1171, "ctx": 4096, "ragged": True, "pad": 5,
         "heads": 32, "kv": 8, "hd": 128, "dims": 128, "halves": False, "page": 64, "typ": "f16", "pool": "f16",
         "salt": 3},
        # one sequence decoding at the benchmark's 8192 positions: latency
        {"name": "attn decode 1 x 8192", "op": "attn", "batch": 1, "new": 1, "ctx": 8192, "ragged": False, "pad": 0,
         "heads": 32, "kv": 8, "hd": 128, "page": 16, "typ": "f16", "salt": 4},
        # 64 sequences decoding at lengths of their own: the cache's bytes
        {"name": "attn decode 64 ragged", "op": "attn", "batch": 64, "new": 1, "ctx": 8192, "ragged": True, "pad": 0,
         "heads": 32, "kv": 8, "hd": 128, "page": 64, "typ": "bf16", "salt": 5},
        # a continuous batch: prompt chunks of odd lengths beside single tokens, the 1B shape
        {"name": "attn mixed 12 hd 64", "op": "attn", "batch": 12, "new": 333, "ctx": 4096, "ragged": True, "pad": 2,
         "heads": 32, "kv": 8, "hd": 64, "page": 32, "typ": "bf16", "salt": 6},
        # the engine's prompt chunk late in a long prompt
        {"name": "attn chunk 512 at 8192", "op": "attn", "batch": 1, "new": 512, "ctx": 8704, "ragged": False, "pad": 0,
         "heads": 32, "kv": 8, "hd": 128, "page": 16, "typ": "f16", "salt": 7},
        # a large chunk of a long document, the 70B shape
        {"name": "attn chunk 2048 at 14336", "op": "attn", "batch": 1, "new": 2048, "ctx": 16384, "ragged": False,
         "pad": 0, "heads": 64, "kv": 8, "hd": 128, "page": 64, "typ": "f16", "salt": 8},
        # the float32 cache: a short chunk of the 1B shape
        {"name": "attn float32 chunk 160", "op": "attn", "batch": 2, "new": 160, "ctx": 2048, "ragged": True, "pad": 0,
         "heads": 32, "kv": 8, "hd": 64, "page": 16, "typ": "f32", "salt": 9},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(32, 8), (28, 4), (64, 8), (8, 8), (12, 2), (71, 1), (6, 2)]


def draw(rng):
    op = rng.choice(["norm", "append", "attn", "attn"])
    heads, kv = rng.choice(HEADS)
    salt = rng.randrange(1 << 30)
    if op == "norm":
        hd = rng.choice([64, 80, 96, 128, 128, 256])
        typ = rng.choice(["f32", "f16", "bf16"])
        out = rng.choice(["f32", "f16", "bf16"]) if typ == "f32" else typ
        most = 8192 * 72 * 128 * 2 // ((heads + kv) * hd * max(BYTES[typ], BYTES[out]))
        return {"op": op, "rows": _log(rng, 1, min(8192, most)), "heads": heads, "kv": kv, "hd": hd,
                "dims": rng.choice([hd, hd, hd // 32 * 16]), "halves": rng.random() < 0.5, "typ": typ, "out": out,
                "far": _log(rng, 16, 131072), "salt": salt}
    if op == "append":
        hd = rng.choice([64, 80, 128, 128])
        typ = rng.choice(["f32", "f16", "bf16"])
        pool = rng.choice(["f16", "f32"]) if typ == "f32" else typ
        batch = _log(rng, 1, 64)
        most = max(1, 8192 * 48 * 128 * 2 // ((heads + 2 * kv) * hd * max(BYTES[typ], BYTES[pool]) * batch))
        new = _log(rng, 1, min(1200, most))
        return {"op": op, "batch": batch, "new": new, "ctx": new + _log(rng, 1, 2048), "ragged": rng.random() < 0.7,
                "pad": rng.choice([0, 0, 7]), "heads": heads, "kv": kv, "hd": hd,
                "dims": rng.choice([0, hd, hd, hd // 32 * 16]), "halves": rng.random() < 0.5,
                "page": rng.choice([16, 32, 64, 24, 1, 256]), "typ": typ, "pool": pool, "salt": salt}
    hd = rng.choice([64, 96, 128, 128])
    typ = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    batch = _log(rng, 1, 64)
    new = 1 if rng.random() < 0.35 else _log(rng, 2, 1024)
    if typ == "f32":
        batch, new = min(batch, 8), min(new, 160)
    # at most 2^29 scores of the padded batch, 2^27 in float32
    most = (1 << (27 if typ == "f32" else 29)) // (batch * heads)
    new = min(new, math.isqrt(most))
    ctx = max(new, _log(rng, 1, min(16384, most // new)))
    while batch * ctx * kv * hd * 2 * BYTES[typ] > 1 << 30:
        batch = max(1, batch // 2)
        ctx = max(new, ctx * 3 // 4)
    return {"op": op, "batch": batch, "new": new, "ctx": ctx, "ragged": rng.random() < 0.7, "pad": rng.choice([0, 0, 5]),
            "heads": heads, "kv": kv, "hd": hd, "page": rng.choice([16, 32, 64, 24, 16, 256]), "typ": typ, "salt": salt}


def _lengths(case):
    """(new rows, positions with them) of each sequence: all alike, or where ragged up to the case's figures, one
    of them at each and some sequences of a mixed batch at a single row."""
    batch, new, ctx = case["batch"], case["new"], case["ctx"]
    if not case["ragged"]:
        return [new] * batch, [ctx] * batch
    r = random.Random(case["salt"])
    n = [new if b == 0 else r.randint(1, new) if b % 3 else max(1, new // (1 + r.randrange(8))) for b in range(batch)]
    if case["op"] == "attn" and new > 1:
        n = [1 if b % 4 == 3 else v for b, v in enumerate(n)]
    kv = [ctx if b == batch - 1 else max(n[b], r.randint(max(1, ctx // 8), ctx)) for b in range(batch)]
    return n, kv


# ---- inputs ------------------------------------------------------------------


def _gb():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gollama.cu_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import gollama_b200

    return gollama_b200


def _normal(shape, g, typ, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES[typ])


def _weights(hd, g):
    return 1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda")


_handle = None


def _kernels(gb):
    """The program's kernel handle, as it keeps one for its life."""
    global _handle
    if _handle is None:
        _handle = gb.Kernels(torch.cuda.current_device())
    return _handle


BASE, EPS = 500000.0, 1e-5


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "norm":
        n = case["rows"]
        # a fused projection's rows: queries, keys, values side by side
        s["qkv"] = _normal((n, (h + 2 * kv) * hd), g, case["typ"], 1.5)
        s["pos"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda", dtype=torch.int32)
        s["wq"], s["wk"] = _weights(hd, g), _weights(hd, g)
        s["q_out"] = torch.zeros((n, h * hd), device="cuda", dtype=TYPES[case["out"]])
        s["k_out"] = torch.zeros((n, kv * hd), device="cuda", dtype=TYPES[case["out"]])
        if own:
            gb = _gb()
            s["gb"], s["kernels"] = gb, _kernels(gb)
            s["norm"], s["rope"] = gb.qk_norm(s["wq"], s["wk"], EPS), gb.rope(BASE, case["dims"], case["halves"])
        return s
    new, lens = _lengths(case)
    page, batch = case["page"], case["batch"]
    pages = [-(-v // page) for v in lens]
    s["max_pages"], s["n_pages"] = max(pages), sum(pages) + 2
    order = torch.randperm(s["n_pages"], generator=g, device="cuda").to(torch.int32)
    table = torch.full((batch, s["max_pages"]), -1, dtype=torch.int32)
    at = 0
    where = torch.full((batch, s["max_pages"]), -1, dtype=torch.int64)
    for b, p in enumerate(pages):
        where[b, :p] = torch.arange(at, at + p)
        at += p
    table = torch.where(where.cuda() >= 0, order[where.clamp(min=0).cuda()], table.cuda())
    s["table"] = table.contiguous()
    s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["q_start"] = torch.tensor([0] + [sum(new[:b + 1]) for b in range(batch)], dtype=torch.int32, device="cuda")
    s["rows"], s["most_new"] = sum(new) + case["pad"], max(new)
    pool = case["pool"] if case["op"] == "append" else case["typ"]
    shape = (s["n_pages"], kv, page, hd)
    s["k_pool"], s["v_pool"] = _normal(shape, g, pool), _normal(shape, g, pool)
    if case["op"] == "append":
        s["qkv"] = _normal((s["rows"], (h + 2 * kv) * hd), g, case["typ"])
        s["q_out"] = torch.zeros((s["rows"], h * hd), device="cuda", dtype=TYPES[pool])
    else:
        # queries and keys of a trained head: a few positions stand out
        s["q"] = _normal((s["rows"], h * hd), g, case["typ"], 2.0)
        s["out"] = torch.zeros_like(s["q"])
    if own:
        gb = _gb()
        s["gb"], s["kernels"] = gb, _kernels(gb)
        s["chunk"] = gb.paged_chunk(s["rows"], batch, s["q_start"], s["kv_lens"], s["table"], s["max_pages"],
                                    s["n_pages"], page, kv, hd, getattr(gb, pool.upper()), s["k_pool"], s["v_pool"])
        if case["op"] == "append":
            s["rope"] = gb.rope(BASE, case["dims"], case["halves"])
    return s


# ---- one pass ----------------------------------------------------------------


def _angles(pos, dims):
    j = torch.arange(dims // 2, device=pos.device, dtype=torch.float64)
    t = pos.double()[:, None] * torch.exp(j * (-2.0 / dims * math.log(BASE)))
    return t.cos().float(), t.sin().float()


def _rotate(x, pos, dims, halves):
    """x [rows][heads][hd] in 32 bits, its first dims rotated at pos [rows]."""
    if not dims:
        return x
    c, n = (v[:, None, :] for v in _angles(pos, dims))
    if halves:
        a, b = x[..., :dims // 2], x[..., dims // 2:dims]
        y = torch.cat((a * c - b * n, a * n + b * c), -1)
    else:
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
        y = torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)
    return torch.cat((y, x[..., dims:]), -1)


def _rows_of(s):
    """For every row: whether it belongs to a sequence, the sequence, its place among the new rows, its position."""
    t = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["q_start"], t, right=True) - 1
    mine = b < s["batch"]
    b = b.clamp(max=s["batch"] - 1)
    first, n = s["q_start"][b], s["q_start"][b + 1] - s["q_start"][b]
    return mine, b, (t - first).long(), (s["kv_lens"][b] - n + t - first).long()


def _norm(s):
    h, kv, hd, n = s["heads"], s["kv"], s["hd"], s["rows"]
    x = s["qkv"].float()
    out = []
    for at, many, w, o in ((0, h, s["wq"], s["q_out"]), (h, kv, s["wk"], s["k_out"])):
        y = x[:, at * hd:(at + many) * hd].reshape(n, many, hd)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        o.copy_(_rotate(y, s["pos"], s["dims"], s["halves"]).reshape(n, many * hd))
        out.append(o)
    return {"q": out[0], "k": out[1]}


def _append(s):
    h, kv, hd, n = s["heads"], s["kv"], s["hd"], s["rows"]
    mine, b, _, pos = _rows_of(s)
    x = s["qkv"].float().reshape(n, h + 2 * kv, hd)
    y = _rotate(x[:, :h + kv], pos, s["dims"], s["halves"])
    s["q_out"].copy_(torch.where(mine[:, None], y[:, :h].reshape(n, h * hd), s["q_out"].float()))
    b, pos, y, v = b[mine], pos[mine], y[mine], x[mine, h + kv:]
    page, slot = s["table"][b, pos // s["page"]].long(), pos % s["page"]
    s["k_pool"][page, :, slot] = y[:, h:].to(s["k_pool"].dtype)
    s["v_pool"][page, :, slot] = v.to(s["v_pool"].dtype)
    return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _attn(s):
    h, kv, hd, n, batch, most = s["heads"], s["kv"], s["hd"], s["rows"], s["batch"], s["most_new"]
    group, L = h // kv, s["max_pages"] * s["page"]
    mine, b, i, _ = _rows_of(s)
    flat = (b * most + i)[mine]
    q = torch.zeros((batch * most, h * hd), device="cuda")
    q[flat] = s["q"][mine].float()
    q = q.reshape(batch, most, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * most, hd)
    at = s["table"].clamp(min=0).long()
    k, v = (p[at].permute(0, 2, 1, 3, 4).reshape(batch, kv, L, hd).float() for p in (s["k_pool"], s["v_pool"]))
    p = torch.arange(L, device="cuda")
    held = p[None, :] < s["kv_lens"][:, None]
    v = torch.where(held[:, None, :, None], v, torch.zeros((), device="cuda"))
    news = s["q_start"][1:] - s["q_start"][:-1]
    last = (s["kv_lens"] - news)[:, None] + torch.arange(most, device="cuda")[None, :]
    seen = (p[None, None, :] <= last[:, :, None]) & held[:, None, :]
    w = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(hd)).reshape(batch, kv, group, most, L)
    w = w.masked_fill_(~seen[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = w.sum(-1, keepdim=True)
    o = w.reshape(batch, kv, group * most, L) @ v
    o = o.reshape(batch, kv, group, most, hd) / torch.where(total > 0, total, torch.ones_like(total))
    o = o.permute(0, 3, 1, 2, 4).reshape(batch * most, h * hd)
    s["out"][mine] = o[flat].to(s["out"].dtype)
    return s["out"]


def run(s):
    h, kv, hd = s["heads"], s["kv"], s["hd"]
    if not own:
        return _norm(s) if s["op"] == "norm" else _append(s) if s["op"] == "append" else _attn(s)
    gb, K = s["gb"], s["kernels"]
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "attn":
        K.attn_chunk_paged(s["chunk"], s["q"], h * hd, h, 1.0 / math.sqrt(hd), s["out"], h * hd, stream=stream)
        return s["out"]
    at, wide, size = s["qkv"].data_ptr(), (h + 2 * kv) * hd, BYTES[s["typ"]] * hd
    q, k, v = at, at + h * size, at + (h + kv) * size
    typ = getattr(gb, s["typ"].upper())
    if s["op"] == "norm":
        K.qk_norm_rope(typ, q, wide, h, k, wide, kv, s["rows"], hd, s["norm"], s["rope"], s["pos"],
                       getattr(gb, s["out"].upper()), s["q_out"], h * hd, s["k_out"], kv * hd, stream=stream)
        return {"q": s["q_out"], "k": s["k_out"]}
    K.rope_append_paged(s["chunk"], typ, q, wide, h, k, wide, v, wide, s["rope"], s["q_out"], h * hd, stream=stream)
    return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "norm":
        values = case["rows"] * (h + kv) * hd
        return {"bytes": values * (BYTES[case["typ"]] + BYTES[case["out"]]) + 4 * case["rows"] + 8 * hd,
                "flops": values * 7}
    new, lens = _lengths(case)
    if case["op"] == "append":
        values = sum(new) * (h + 2 * kv) * hd
        return {"bytes": values * (BYTES[case["typ"]] + BYTES[case["pool"]]) + 4 * sum(-(-v // case["page"]) for v in lens),
                "flops": sum(new) * (h + kv) * hd * 3}
    size = BYTES[case["typ"]]
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, lens))
    return {"bytes": size * hd * (2 * h * sum(new) + 2 * kv * sum(lens)) + 4 * sum(-(-v // case["page"]) for v in lens),
            "flops": 4 * hd * h * seen}


# ---- the definitions in 64 bits ----------------------------------------------


def _turned(x, pos, dims, halves):
    """x [rows][heads][hd] float64, each pair taken as a complex number and turned by its angle."""
    x = x.clone()
    if dims:
        j = torch.arange(0, dims, 2, device=x.device, dtype=torch.float64)
        angle = pos.double()[:, None, None] * torch.pow(torch.full_like(j, BASE), -j / dims)
        turn = torch.polar(torch.ones_like(angle), angle)
        i = torch.arange(dims // 2, device=x.device)
        lo, hi = (i, i + dims // 2) if halves else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., lo], x[..., hi]) * turn
        x[..., lo], x[..., hi] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    if case["op"] == "norm":
        x = s["qkv"].double().reshape(case["rows"], h + 2 * kv, hd)
        got = {}
        for name, y, w in (("q", x[:, :h], s["wq"]), ("k", x[:, h:h + kv], s["wk"])):
            y = y / ((y * y).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
            got[name] = _turned(y, s["pos"], case["dims"], case["halves"]).reshape(case["rows"], -1)
        return got
    new, lens = _lengths(case)
    page = case["page"]
    slots = []  # each sequence's positions as rows of the pool's (page, slot) plane
    for b, L in enumerate(lens):
        p = torch.arange(L, device="cuda")
        slots.append((s["table"][b].long()[p // page], p % page))
    if case["op"] == "append":
        x = s["qkv"].double().reshape(s["rows"], h + 2 * kv, hd)
        q, kp, vp = s["q_out"].double(), s["k_pool"].double(), s["v_pool"].double()
        at = 0
        for b, (n, L) in enumerate(zip(new, lens)):
            y = _turned(x[at:at + n, :h + kv], torch.arange(L - n, L, device="cuda"), case["dims"], case["halves"])
            pages, slot = slots[b][0][L - n:], slots[b][1][L - n:]
            q[at:at + n] = y[:, :h].reshape(n, h * hd)
            kp[pages, :, slot] = y[:, h:]
            vp[pages, :, slot] = x[at:at + n, h + kv:]
            at += n
        return {"q": q, "k_pool": kp, "v_pool": vp}
    out, group, at = s["out"].double(), h // kv, 0
    for b, (n, L) in enumerate(zip(new, lens)):
        pages, slot = slots[b]
        k, v = s["k_pool"][pages, :, slot].double(), s["v_pool"][pages, :, slot].double()  # [L][kv][hd]
        q = s["q"][at:at + n].double().reshape(n, kv, group, hd)
        after = torch.arange(L, device="cuda")[None, :] > torch.arange(L - n, L, device="cuda")[:, None]
        for c in range(kv):
            w = torch.einsum("ngd,ld->ngl", q[:, c], k[:, c]) / math.sqrt(hd)
            w = torch.softmax(w.masked_fill_(after[:, None, :], -math.inf), -1)
            out[at:at + n, c * group * hd:(c + 1) * group * hd] = torch.einsum("ngl,ld->ngd", w, v[:, c]).reshape(n, -1)
        at += n
    return out
