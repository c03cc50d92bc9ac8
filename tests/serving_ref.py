"""Plain 64-bit forms of the serving-step operators (per-head norms and
rotation, the paged append, attention of new rows over the pages), and batches
to try them on. Reference arithmetic: cpu.RoPE (backend/cpu/cpu.go:118) and
cpu.AttnDecode (backend/cpu/cpu.go:140), one row at a time."""
import numpy as np
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(typ: str) -> float:
    """The largest relative error of one rounding to the type."""
    return torch.finfo(DT[typ]).eps / 2


def rotate(x, pos, dims, halves, base, freq=None):
    """x [rows][heads][hd] float64, its first dims turned at pos[rows]."""
    x = x.clone()
    if not dims:
        return x
    j = torch.arange(dims // 2, dtype=torch.float64, device=x.device)
    t = pos.double()[:, None] * base ** (-2.0 * j / dims)
    if freq is not None:
        t = t / freq.double()
    c, s = t.cos()[:, None], t.sin()[:, None]
    lo, hi = (slice(0, dims // 2), slice(dims // 2, dims)) if halves else (slice(0, dims, 2), slice(1, dims, 2))
    a, b = x[..., lo].clone(), x[..., hi].clone()
    x[..., lo], x[..., hi] = a * c - b * s, a * s + b * c
    return x


def norm(x, w, eps):
    return x if w is None else x * w.double() / (x.square().mean(-1, keepdim=True) + eps).sqrt()


class Batch:
    """Sequences of (new rows, positions with them) over a shuffled page pool; `first` rows before the first
    sequence and `pad` behind the last belong to none."""

    def __init__(self, seqs, n_kv, hd, page, typ, seed, first=0, pad=0, spare_pages=2, wide_table=1):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.n_kv, self.hd, self.page, self.typ = seqs, n_kv, hd, page, typ
        self.batch = len(seqs)
        pages = [max(0, -(-kv // page)) for _, kv in seqs]
        self.max_pages, self.n_pages = max(pages + [0]) + wide_table, sum(pages) + spare_pages
        order = torch.randperm(self.n_pages, generator=g)
        table = torch.full((self.batch, self.max_pages), -1, dtype=torch.int32)
        at = 0
        for b, p in enumerate(pages):
            table[b, :p] = order[at:at + p].int()
            at += p
        starts = np.cumsum([first] + [n for n, _ in seqs])
        self.rows = int(starts[-1]) + pad
        self.table = table.cuda()
        self.q_start = torch.tensor(starts, dtype=torch.int32).cuda()
        self.kv_lens = torch.tensor([kv for _, kv in seqs], dtype=torch.int32).cuda()
        self.starts = [int(v) for v in starts]
        shape = (self.n_pages, n_kv, page, hd)
        self.k = torch.randn(shape, generator=g).to(DT[typ]).cuda()
        self.v = torch.randn(shape, generator=g).to(DT[typ]).cuda()

    def slots(self, b, lo, hi):
        """Physical page and slot of positions [lo, hi) of sequence b."""
        p = torch.arange(lo, hi, device="cuda")
        return self.table[b].long()[p // self.page], p % self.page

    def chunk(self, gb):
        return gb.paged_chunk(self.rows, self.batch, self.q_start, self.kv_lens, self.table, self.max_pages,
                              self.n_pages, self.page, self.n_kv, self.hd, getattr(gb, self.typ.upper()), self.k, self.v)

    def attention(self, q, n_heads, scale, out):
        """(outputs, sum of p |v|, largest |q||k| scale) in float64; rows of no sequence as in `out`."""
        o, mag, big = out.double().clone(), torch.zeros_like(out, dtype=torch.float64), 0.0
        group = n_heads // self.n_kv
        for b, (n, kv) in enumerate(self.seqs):
            r0 = self.starts[b]
            if not n:
                continue
            qs = q[r0:r0 + n].double().reshape(n, self.n_kv, group, self.hd)
            pages, slot = self.slots(b, 0, max(kv, 0))
            k, v = self.k[pages, :, slot].double(), self.v[pages, :, slot].double()
            seen = torch.arange(max(kv, 0), device="cuda")[None, :] <= torch.arange(kv - n, kv, device="cuda")[:, None]
            w = torch.einsum("nhgd,lhd->nhgl", qs, k) * scale
            w = torch.where(seen[:, None, None, :], w, -torch.inf)
            p = torch.softmax(w, -1)
            p = torch.where(seen.any(1)[:, None, None, None], p, torch.zeros_like(p))
            v = torch.where(torch.isfinite(v), v, torch.zeros_like(v)) if not torch.isfinite(v).all() else v
            o[r0:r0 + n] = torch.einsum("nhgl,lhd->nhgd", p, v).reshape(n, -1)
            mag[r0:r0 + n] = torch.einsum("nhgl,lhd->nhgd", p, v.abs()).reshape(n, -1)
            if kv > 0:
                lengths = torch.einsum("nhgd,lhd->nhgl", qs.abs(), k.nan_to_num(0, 0, 0).abs())
                big = max(big, float(lengths.max()) * scale)
        return o, mag, big
