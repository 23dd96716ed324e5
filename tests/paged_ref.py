"""Inputs and the 64-bit definition for the paged-cache tests: a cache in any page layout, and
append and attention one token and one key at a time over plain lists of positions."""

import math

import torch

EPS = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


class Setup:
    """A random cache of `lens` positions (the step's `new` tokens included) per sequence, pages
    handed out in no order.  layout "slot": [pages, page, kv, dim]; "head": [pages, kv, page,
    dim] transposed; "padded": pages and slots with gaps between them.  Slots past a sequence's
    length hold NaN.  `shared`: the first positions' whole pages are the same ones for every
    sequence, the copies of an unfull last page hold the same values."""

    def __init__(self, dev, dtype, heads, kv, dim, page, lens, new, seed=0, layout="slot",
                 shared=0, extra_width=1, qscale=2.0):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.dtype, self.heads, self.kv, self.dim, self.page = dev, dtype, heads, kv, dim, page
        self.lens, self.new = list(lens), list(new)
        batch = len(self.lens)
        need = [-(-max(n, 0) // page) for n in self.lens]
        common = shared // page
        pages = common + sum(max(0, n - common) for n in need) + 2
        order = torch.randperm(pages, generator=g).tolist()
        width = max(need + [common]) + extra_width
        self.table = torch.full((batch, width), -1, dtype=torch.int32)
        at = common
        for b in range(batch):
            for i in range(max(need[b], common)):
                if i < common:
                    self.table[b, i] = order[i]
                else:
                    self.table[b, i] = order[at]
                    at += 1
        k = torch.full((pages, page, kv, dim), float("nan"))
        v = torch.full((pages, page, kv, dim), float("nan"))
        pre_k = torch.randn(max(shared, 1), kv, dim, generator=g)
        pre_v = torch.randn(max(shared, 1), kv, dim, generator=g)
        for b in range(batch):
            for j in range(max(self.lens[b], shared)):
                pg, sl = int(self.table[b, j // page]), j % page
                if j < shared:
                    k[pg, sl], v[pg, sl] = pre_k[j], pre_v[j]
                else:
                    k[pg, sl] = torch.randn(kv, dim, generator=g)
                    v[pg, sl] = torch.randn(kv, dim, generator=g)
        self.k, self.v = self._place(k.to(dtype), layout), self._place(v.to(dtype), layout)
        tokens = sum(self.new)
        self.q = (torch.randn(tokens, heads, dim, generator=g) * qscale).to(dtype)
        self.qkv = torch.randn(tokens, (heads + 2 * kv) * dim, generator=g).to(dtype)
        cu = [0]
        for n in self.new:
            cu.append(cu[-1] + n)
        self.starts = cu
        self.cu = torch.tensor(cu, dtype=torch.int32)

    def _place(self, x, layout):
        if layout == "head":
            return x.transpose(1, 2).contiguous().to(self.dev).transpose(1, 2)
        if layout == "padded":
            pages, page, kv, dim = x.shape
            big = torch.full((pages, page + 3, kv + 1, dim + 8), float("nan"), dtype=x.dtype)
            big[:, :page, :kv, :dim] = x
            return big.to(self.dev)[:, :page, :kv, :dim]
        return x.to(self.dev)

    def cache(self, kernels):
        self.table_d = self.table.to(self.dev)
        self.lens_d = torch.tensor(self.lens, dtype=torch.int32, device=self.dev)
        return kernels.PagedKV(self.k, self.v, self.table_d, self.lens_d)

    def cu_d(self):
        return self.cu.to(self.dev)


def key(s, b, j, x):
    """Position j of sequence b in x (k or v, on the CPU), or None where no page holds it."""
    if j >= s.table.shape[1] * s.page:
        return None
    pg = int(s.table[b, j // s.page])
    if pg < 0 or pg >= x.shape[0]:
        return None
    return x[pg, j % s.page]


def attention(s, window=0, sinks=0, shared=0, scale=None):
    """(out, lse, vmax) in float64 from the definition; vmax [tokens, heads] is the largest |v|
    that a row sees."""
    scale = s.dim ** -0.5 if scale is None else scale
    group = s.heads // s.kv
    q, k, v = s.q.double(), s.k.cpu().double(), s.v.cpu().double()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    vmax = torch.zeros(q.shape[:2], dtype=torch.float64)
    for b, (n, total) in enumerate(zip(s.new, s.lens)):
        for i in range(n):
            p = total - n + i
            seen = [j for j in range(p + 1) if not window or j > p - window or j < sinks]
            rows = [(key(s, 0 if j < shared else b, j, k), key(s, 0 if j < shared else b, j, v))
                    for j in seen]
            rows = [r for r in rows if r[0] is not None]
            if not rows:
                continue
            ks, vs = torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])
            t = s.starts[b] + i
            for h in range(s.heads):
                sc = (ks[:, h // group] @ q[t, h]) * scale
                lse[t, h] = torch.logsumexp(sc, 0)
                out[t, h] = torch.exp(sc - lse[t, h]) @ vs[:, h // group]
                vmax[t, h] = vs[:, h // group].abs().max()
    return out, lse, vmax


def append(s, cos, sin, rope_rows=None):
    """(q, k, v) in float64 after the append; cos, sin float tables [positions, dim / 2]."""
    rows = cos.shape[0] if rope_rows is None else rope_rows
    half, c, sn = s.dim // 2, cos.double(), sin.double()
    k, v = s.k.cpu().double().clone(), s.v.cpu().double().clone()
    x = s.qkv.double().view(-1, s.heads + 2 * s.kv, s.dim)
    q = torch.zeros(x.shape[0], s.heads, s.dim, dtype=torch.float64)
    for b, (n, total) in enumerate(zip(s.new, s.lens)):
        for i in range(n):
            p, t = total - n + i, s.starts[b] + i
            if p < 0 or p >= rows:
                continue
            lo, hi = x[t, :, :half], x[t, :, half:]
            rot = torch.cat((lo * c[p] - hi * sn[p], hi * c[p] + lo * sn[p]), -1)
            q[t] = rot[:s.heads]
            dst = key(s, b, p, k)
            if dst is None:
                continue
            dst.copy_(rot[s.heads:s.heads + s.kv])
            key(s, b, p, v).copy_(x[t, s.heads + s.kv:])
    return q, k, v


def close(got, ref, vmax, dtype):
    """Attention's bound.  Per output: its own rounding (half a step of the value), and the
    probabilities', each rounded to the 16-bit type before its product with v: half a step of p
    times |v|, at most vmax half a step in all since they sum to 1, doubled because the sum that
    divides them is of the unrounded ones.  fp32 terms: scores of |s| <= 60 off by 1e-5 relative
    move p by 1e-3 at most (their fp32 sums' rounding, exp's and log2 e's), counted against vmax."""
    e = EPS[dtype]
    bound = ref.abs() * e + (2 * e + 1e-3) * vmax[..., None] + 1e-7
    off = (got.double().cpu() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert (off <= bound).all(), f"largest excess {(off - bound).max():.3e}"
