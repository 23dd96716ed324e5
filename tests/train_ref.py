"""64-bit definitions for the tests of training attention and of dropout, and how far the kernels may
be off by the roundings that they make."""

import math

import numpy as np
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}        # half of the least number's step
U32 = 2.0 ** -24
LOG2E = 1.0 / math.log(2.0)


def hidden(n, window):
    i, j = torch.arange(n)[:, None], torch.arange(n)[None]
    return (j > i) | ((j <= i - window) if window else torch.zeros_like(j > i))


def attention(q, k, v, cu, dout=None, window=0, scale=None):
    """{name: (value, bound)} of out and stats, and of dq, dk, dv with `dout`, all in float64 on the
    CPU.  Values by the formulas; bounds count half a step for each rounding to the type (the
    probabilities, dS, the saved output, the result), an fp32 product's error of D + 8 half steps,
    and for a sum in fp32 as many half steps as it has terms."""
    half, tiny = HALF[q.dtype], TINY[q.dtype]
    q, k, v = q.cpu().double(), k.cpu().double(), v.cpu().double()
    tokens, heads, dim = q.shape
    kv = k.shape[1]
    group = heads // kv
    scale = dim ** -0.5 if scale is None else scale
    z = lambda *s: torch.zeros(s, dtype=torch.float64)  # noqa: E731
    r = {"out": (z(tokens, heads, dim), z(tokens, heads, dim)),
         "stats": (z(tokens, heads, 2), z(tokens, heads, 2)),
         "dq": (z(tokens, heads, dim), z(tokens, heads, dim)),
         "dk": (z(tokens, kv, dim), z(tokens, kv, dim)),
         "dv": (z(tokens, kv, dim), z(tokens, kv, dim))}
    if dout is not None:
        dout = dout.cpu().double()
    prod = (dim + 8) * U32
    for t0, t1 in zip(cu, cu[1:]):
        n = t1 - t0
        if n <= 0:
            continue
        off = hidden(n, window)
        sums = n * U32
        for h in range(heads):
            g, sl = h // group, slice(t0, t1)
            s = (q[sl, h] @ k[sl, g].t()) * scale
            s = s.masked_fill(off, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            l = p.sum(-1, keepdim=True)
            p = p / l
            # a score's error, and by it a probability's, relative (twice: its own and the maximum's)
            es = ((q[sl, h].abs() @ k[sl, g].abs().t()) * abs(scale) * prod).masked_fill(off, 0).amax(-1, keepdim=True)
            ep = 2 * es + 8 * U32 + sums
            o, oa = p @ v[sl, g], p @ v[sl, g].abs()
            eo = half * o.abs() + (half + ep + sums) * oa + tiny
            r["out"][0][sl, h], r["out"][1][sl, h] = o, eo * 1.01
            r["stats"][0][sl, h] = torch.cat((m * LOG2E, l), -1)
            r["stats"][1][sl, h] = torch.cat(((es + 4 * U32 * m.abs()) * LOG2E, l * ep), -1) * 1.01 + 1e-7
            if dout is None:
                continue
            do = dout[sl, h]
            dp, dpa = do @ v[sl, g].t(), do.abs() @ v[sl, g].abs().t()
            delta = (do * o).sum(-1, keepdim=True)
            ed = (do.abs() * eo).sum(-1, keepdim=True) + prod * (do.abs() * o.abs()).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            # (fp16's dS are scaled so that the largest of its bound is near the type's end: what
            # is lost below its least number is 2^-36 of that bound)
            top = do.norm(dim=-1, keepdim=True).max() * v[sl, g].norm(dim=-1).max()
            eds = ds.abs() * (half + ep) + p * (ed + prod * (dpa + delta.abs())) * 1.01
            eds = eds + (2.0 ** -36 * top if tiny else 0.0)
            eds = eds.masked_fill(off, 0.0)
            ew = (p * (half + ep) + (2.0 ** -40 if tiny else 0.0)).masked_fill(off, 0.0)
            dq = ds @ k[sl, g] * scale
            r["dq"][0][sl, h] = dq
            r["dq"][1][sl, h] = (half * dq.abs() + (eds + sums * ds.abs()) @ k[sl, g].abs() * abs(scale) + tiny) * 1.01
            r["dk"][0][sl, g] += ds.t() @ q[sl, h] * scale
            r["dk"][1][sl, g] += (eds + group * sums * ds.abs()).t() @ q[sl, h].abs() * abs(scale)
            r["dv"][0][sl, g] += p.t() @ do
            r["dv"][1][sl, g] += (ew + group * sums * p).t() @ do.abs()
    for name in ("dk", "dv"):
        val, bound = r[name]
        r[name] = (val, (bound + half * val.abs() + tiny) * 1.01)
    return r


def assert_within(got, ref, what):
    value, bound = ref
    got = got.detach().cpu().double()
    off = (got - value).abs()
    worst = (off / bound.clamp(min=1e-300)).flatten()
    at = int(worst.argmax())
    assert not torch.isnan(got).any(), f"{what}: NaN"
    assert bool((off <= bound).all()), \
        f"{what}: off by {off.flatten()[at]:.3e} at {at}, bound {bound.flatten()[at]:.3e}"


def philox(seed, step, site, groups):
    """The eight 16-bit numbers of each group, [groups, 8], from the generator's definition in whole
    numbers of any size (no wrapped products)."""
    out = np.zeros((len(groups), 8), dtype=np.int64)
    for n, g in enumerate(groups):
        c = [g & 0xFFFFFFFF, g >> 32, step & 0xFFFFFFFF, site]
        key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(10):
            x, y = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(y >> 32) ^ c[1] ^ key[0], y & 0xFFFFFFFF, (x >> 32) ^ c[3] ^ key[1],
                 x & 0xFFFFFFFF]
            key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out[n] = [w >> (16 * h) & 0xFFFF for w in c for h in (0, 1)]
    return out


def kept(seed, step, site, rows, cols, p):
    """bool [rows, cols]: what a site keeps."""
    per = -(-cols // 8)
    u = philox(seed, step, site, range(rows * per)).reshape(rows, per * 8)[:, :cols]
    return torch.from_numpy(u >= math.floor(65536 * p + 0.5))


def drop_scale(p):
    cut = math.floor(65536 * p + 0.5)
    return 65536.0 / (65536 - cut) if cut < 65536 else 0.0
