"""Training attention of a packed batch, forward and backward, against its 64-bit definition."""

import math

import pytest
import torch

from tests import train_ref as ref
from tests.gpu_util import banner

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def make(dev, dtype, heads, kv, dim, lens, pad=0, seed=0, qscale=2.0, gscale=1.0, layout="qkv"):
    """(q, k, v, dout, offsets) on the GPU; layout "qkv": columns of one buffer, "heads": one head
    behind the other, "plain": tensors of their own."""
    g = torch.Generator().manual_seed(seed)
    tokens = sum(lens) + pad
    x = torch.randn(tokens, heads + 2 * kv, dim, generator=g)
    x[:, :heads] *= qscale
    x = x.to(dtype)
    parts = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if layout == "qkv":
        x = x.to(dev)
        q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    elif layout == "heads":
        q, k, v = (t.transpose(0, 1).contiguous().to(dev).transpose(0, 1) for t in parts)
    else:
        q, k, v = (t.contiguous().to(dev) for t in parts)
    dout = (torch.randn(tokens, heads, dim, generator=g) * gscale).to(dtype).to(dev)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return q, k, v, dout, cu


def run(q, k, v, dout, cu, **kw):
    from solution import kernels

    c = torch.tensor(cu, dtype=torch.int32, device=q.device) if cu is not None else None
    out, stats = kernels.attention_fwd(q, k, v, c, **kw)
    grads = kernels.attention_bwd(dout, q, k, v, out, stats, c, **kw)
    torch.cuda.synchronize()
    return dict(zip(("out", "stats", "dq", "dk", "dv"), (out, stats, *grads)))


def check(got, q, k, v, dout, cu, **kw):
    kw.pop("max_len", None)
    want = ref.attention(q, k, v, cu if cu is not None else [0, q.shape[0]], dout, **kw)
    for name in ("out", "stats", "dq", "dk", "dv"):
        ref.assert_within(got[name], want[name], name)


CASES = [
    # dtype, heads, kv, dim, lens, pad, window, layout
    (F16, 1, 1, 64, (1,), 0, 0, "plain"),
    (BF16, 2, 1, 128, (1,), 0, 0, "qkv"),
    (F16, 2, 2, 64, (2, 1, 3), 0, 0, "plain"),
    (BF16, 12, 2, 128, (17,), 0, 0, "qkv"),
    (F16, 4, 4, 64, (63, 64, 65), 0, 0, "qkv"),
    (BF16, 4, 2, 128, (127, 1, 128, 129), 5, 0, "heads"),
    (F16, 6, 2, 128, (200, 0, 0, 57, 300), 70, 0, "qkv"),
    (BF16, 14, 2, 64, (333, 90), 0, 0, "qkv"),
    (F16, 2, 1, 128, (700,), 0, 0, "plain"),
    (BF16, 2, 1, 64, (700, 333), 140, 0, "heads"),
    (F16, 2, 1, 128, (300, 41), 3, 1, "qkv"),
    (BF16, 2, 1, 64, (300, 41), 3, 2, "qkv"),
    (F16, 4, 2, 64, (500, 260), 0, 63, "qkv"),
    (BF16, 4, 2, 128, (500, 260), 9, 64, "heads"),
    (F16, 3, 1, 128, (450,), 0, 129, "qkv"),
    (BF16, 3, 3, 64, (450, 450), 0, 300, "plain"),
    (F16, 2, 2, 64, tuple([3, 1, 0, 2] * 40), 200, 0, "qkv"),
]


@pytest.mark.parametrize("dtype,heads,kv,dim,lens,pad,window,layout", CASES)
def test_definition(cuda, dtype, heads, kv, dim, lens, pad, window, layout):
    banner("attention", dtype, heads, kv, dim, lens, pad, window, layout)
    q, k, v, dout, cu = make(cuda, dtype, heads, kv, dim, lens, pad, seed=3, layout=layout)
    got = run(q, k, v, dout, cu, window=window, max_len=max(lens))
    check(got, q, k, v, dout, cu, window=window)
    tail = sum(lens)
    for name in ("out", "stats", "dq", "dk", "dv"):  # rows of no sequence
        assert not got[name][tail:].any(), name


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens,window", [((1500,), 0), ((1100, 900), 400)])
def test_long(cuda, dtype, lens, window):
    banner("long", dtype, lens, window)
    q, k, v, dout, cu = make(cuda, dtype, 6, 2, 128, lens, 30, seed=4)
    check(run(q, k, v, dout, cu, window=window), q, k, v, dout, cu, window=window)


def test_one_sequence_without_offsets(cuda):
    q, k, v, dout, _ = make(cuda, F16, 4, 2, 64, (150,), seed=5)
    check(run(q, k, v, dout, None), q, k, v, dout, None)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.125, 0.4, 1e-30])
def test_scales(cuda, dtype, scale):
    q, k, v, dout, cu = make(cuda, dtype, 2, 1, 64, (90, 40), seed=6)
    check(run(q, k, v, dout, cu, scale=scale), q, k, v, dout, cu, scale=scale)


@pytest.mark.parametrize("gscale", [1e-4, 3e3])
def test_gradients_of_any_size_in_fp16(cuda, gscale):
    """The scale of a loss: dS of 1e-8 and of 1e5 have their bits (a plain fp16 of them has none)."""
    q, k, v, dout, cu = make(cuda, F16, 4, 2, 128, (300,), seed=7, gscale=gscale)
    if gscale > 1:
        q, k = q * 0.125, k * 0.125
        v = v * 0.25
    check(run(q, k, v, dout, cu), q, k, v, dout, cu)


def test_max_len_chooses_no_result(cuda):
    q, k, v, dout, cu = make(cuda, BF16, 4, 2, 128, (400, 130), seed=8)
    for n in (0, 1, 400, 100000):
        check(run(q, k, v, dout, cu, max_len=n), q, k, v, dout, cu)


def test_results_do_not_depend_on_timing(cuda):
    q, k, v, dout, cu = make(cuda, F16, 12, 2, 128, (900, 300), seed=9)
    a = run(q, k, v, dout, cu)
    for _ in range(3):
        b = run(q, k, v, dout, cu)
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("what", ["v", "k", "q", "dout"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_not_finite_stays_with_those_who_see_it(cuda, dtype, what, value):
    """An infinity or NaN in one sequence's row leaves the other sequences, and in k and v the rows
    before it, as they are without it."""
    banner("not finite", dtype, what, value)
    q, k, v, dout, cu = make(cuda, dtype, 4, 2, 64, (50, 70, 40), seed=10, layout="plain")
    want = ref.attention(q, k, v, cu, dout)
    at = 50 + 33
    {"q": q, "k": k, "v": v, "dout": dout}[what][at, -1, 5] = value
    got = run(q, k, v, dout, cu)
    for name in ("out", "stats", "dq", "dk", "dv"):
        for s in (slice(0, 50), slice(120, 160)):
            ref.assert_within(got[name][s], tuple(t[s] for t in want[name]), name)
    # its own sequence's rows before it see none of it
    for name in ("out", "stats", "dq"):
        ref.assert_within(got[name][50:at], tuple(t[50:at] for t in want[name]), name)
    # nor do the keys behind it, where it is a row's
    if what in ("q", "dout"):
        for name in ("dk", "dv"):
            ref.assert_within(got[name][at + 1:120], tuple(t[at + 1:120] for t in want[name]), name)
    # and what is touched says so
    touched = {"v": ("out", "dq", "dk"), "k": ("out", "dq", "dk"), "q": ("out", "dq", "dk", "dv"),
               "dout": ("dq", "dk", "dv")}[what]
    if math.isnan(value):
        for name in touched:
            assert torch.isnan(got[name][50:120].float()).any(), name


def test_gradient_against_differences(cuda):
    """(L(x + h d) - L(x - h d)) / 2h = <gradient, d> with L = sum(out * w), by the kernel's forward
    pass alone: fp16 outputs are off by half a step each, which the sum over them averages."""
    q, k, v, dout, cu = make(cuda, F16, 4, 2, 64, (120, 60), seed=11, qscale=1.0, layout="plain")
    from solution import kernels

    got = run(q, k, v, dout, cu)
    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(12)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        h = 2.0 ** -4
        d = torch.randint(-1, 2, x.shape, generator=g).to(x)  # x +- h d: exact but for x's step
        up, down = x + h * d, x - h * d
        step = (up.double() - down.double())

        def loss(y):
            args = {"dq": (y, k, v), "dk": (q, y, v), "dv": (q, k, y)}[name]
            return kernels.attention_fwd(*args, c)[0].double()

        a, b = loss(up), loss(down)
        moved = ((a - b) * dout.double()).sum()
        told = (got[name].double() * step).sum()
        # roundings of a and b: independent, half a step at most each (their mean square a third of
        # that, six of the sum's deviations); the third-order term h^2 / 6 of the softmax's change
        noise = 6 * ((2.0 ** -11 * dout.double()) ** 2 * (a ** 2 + b ** 2) / 3).sum().sqrt()
        third = 0.02 * (got[name].double().norm() * step.norm()) / 4
        assert (moved - told).abs() <= noise + third, (name, float(moved), float(told), float(noise))


def test_written_views(cuda):
    """Gradients into the columns of one buffer, beside columns that stay as they are."""
    from solution import kernels

    q, k, v, dout, cu = make(cuda, BF16, 4, 2, 64, (90, 30), pad=6, seed=13)
    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    out, stats = kernels.attention_fwd(q, k, v, c)
    big = torch.full((126, 10, 64), 7.0, dtype=BF16, device=cuda)
    kernels.attention_bwd(dout, q, k, v, out, stats, c, grads=(big[:, 1:5], big[:, 5:7], big[:, 8:10]))
    plain = kernels.attention_bwd(dout, q, k, v, out, stats, c)
    assert torch.equal(big[:, 1:5], plain[0]) and torch.equal(big[:, 5:7], plain[1])
    assert torch.equal(big[:, 8:10], plain[2])
    assert (big[:, 0] == 7).all() and (big[:, 7] == 7).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("value", [math.nan, math.inf, 6e4])
def test_what_lies_in_rows_of_no_sequence_does_not_matter(cuda, dtype, value):
    """Rows of padding that hold NaN, infinities or large numbers, as memory that nothing wrote does."""
    banner("padding", dtype, value)
    q, k, v, dout, cu = make(cuda, dtype, 4, 2, 64, (150, 40), pad=60, seed=14, layout="plain")
    clean = run(q, k, v, dout, cu)
    for t in (q, k, v, dout):
        t[190:] = value
    got = run(q, k, v, dout, cu)
    assert all(torch.equal(got[n], clean[n]) for n in clean)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_gradients_that_are_not_finite(cuda, dtype):
    """A loss whose scale was too high: a row whose dout holds an infinity or NaN has NaN for its dq, and so
    have all dk and dv that it sees; nothing else has."""
    q, k, v, dout, cu = make(cuda, dtype, 4, 2, 64, (200, 90), seed=15, layout="plain")
    want = ref.attention(q, k, v, cu, dout)
    for value in (math.inf, math.nan):
        d = dout.clone()
        d[120, 1, 7] = value  # head 1 reads key head 0
        got = run(q, k, v, d, cu)
        assert torch.isnan(got["dq"][120, 1]).all()
        for name in ("dk", "dv"):
            assert torch.isnan(got[name][:121, 0]).all()
            ref.assert_within(got[name][121:], tuple(t[121:] for t in want[name]), name)
            ref.assert_within(got[name][:, 1], tuple(t[:, 1] for t in want[name]), name)
        rest = torch.ones(290, 4, dtype=torch.bool)
        rest[120, 1] = False
        ref.assert_within(got["dq"].cpu()[rest], tuple(t[rest] for t in want["dq"]), "dq")
    got = run(q, k, v, torch.full_like(dout, math.nan), cu)
    assert all(torch.isnan(got[n]).all() for n in ("dq", "dk", "dv"))


def test_scores_that_are_not_finite(cuda):
    """Keys with a score of -inf have no weight beside others; a row with such keys only, or with one of
    +inf, is NaN, as the formula is."""
    q, k, v, dout, cu = make(cuda, BF16, 1, 1, 64, (300,), seed=16, layout="plain")
    q[:, 0, 0], k[:, 0, 0] = -1.0, 0.0
    k[0, 0, 0] = math.inf
    out = run(q, k, v, dout, cu)
    q1 = q[1:], k[1:], v[1:]
    want = ref.attention(*q1, [0, 299])
    assert torch.isnan(out["out"][0]).all()
    for name in ("out", "stats"):
        ref.assert_within(out[name][1:], want[name], name)
    q[150, 0, 0] = 1.0
    out = run(q, k, v, dout, cu)
    assert torch.isnan(out["out"][150]).all() and not torch.isnan(out["out"][149]).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_of_any_size(cuda, dtype):
    """Scores of 1e5 and more, whose statistics no float holds to a step of 1: rows that see one key have a
    probability of 1, whatever its score."""
    q, k, v, dout, cu = make(cuda, dtype, 2, 1, 64, (1,) * 40, seed=17, qscale=60.0, layout="plain")
    for scale in (1e3, 1e9, -1e9, 1e30):
        got = run(q, k, v, dout, cu, scale=scale)
        # The maximum as a float is off by up to 2^-5 where it is near 2^20, the row's sum 2^that, and so is its
        # one probability before the division; that is rounded to the type, the sum is not, and the quotient
        # is rounded again: two half steps.
        away = (got["out"].double() - v.double()).abs()
        assert (away <= 2.01 * ref.HALF[dtype] * v.double().abs()).all()
        sums = dout.double().sum(1, keepdim=True)
        off = (got["dv"].double() - sums).abs()
        assert (off <= ref.HALF[dtype] * sums.abs() + 2.0 ** -20).all()
        # (dS is 0 but for the saved output's half step: up to 2^-11 of sum |do v|, 0.03 here; with a scale of
        # 1e9 and q of 60 that is 2e9, beyond fp16's largest number: infinite there, but no NaN)
        assert not torch.isnan(got["dq"]).any() and not torch.isnan(got["dk"]).any()


def test_nothing_to_do(cuda):
    from solution import kernels

    e = torch.empty(0, 4, 64, dtype=F16, device=cuda)
    k = torch.empty(0, 2, 64, dtype=F16, device=cuda)
    cu = torch.zeros(1, dtype=torch.int32, device=cuda)
    for c in (None, cu):
        out, stats = kernels.attention_fwd(e, k, k, c)
        assert out.shape == (0, 4, 64) and stats.shape == (0, 4, 2)
        assert [t.shape[0] for t in kernels.attention_bwd(out, e, k, k, out, stats, c)] == [0, 0, 0]
    q, k, v, dout, _ = make(cuda, F16, 4, 2, 64, (), pad=70, seed=18)
    got = run(q, k, v, dout, [0])  # rows, and no sequence
    assert not any(t.any() for t in got.values())


def test_offsets_past_32_bits(cuda):
    """Heads 2^31 + 64 elements apart."""
    q, k, v, dout, cu = make(cuda, F16, 2, 2, 64, (100, 29), seed=19, layout="plain")
    far = (1 << 31) + 64
    big = torch.empty(far + 129 * 64, dtype=F16, device=cuda)

    def place(t):
        x = torch.as_strided(big, t.shape, (64, far, 1))
        x.copy_(t)
        return x

    clean = run(q, k, v, dout, cu)
    for i in range(4):  # (one at a time: they share the memory)
        args = [q, k, v, dout]
        args[i] = place(args[i])
        got = run(*args, cu)
        assert all(torch.equal(got[n], clean[n]) for n in clean)
    from solution import kernels

    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    grads = torch.as_strided(big, (129, 2, 64), (64, far, 1)), torch.empty_like(k), torch.empty_like(v)
    got = kernels.attention_bwd(dout, q, k, v, clean["out"], clean["stats"], c, grads=grads)
    assert torch.equal(got[0], clean["dq"])


def test_many_sequences_and_one_among_empty_ones(cuda):
    """More offsets than a wave holds, and more empty sequences in a row than it looks through."""
    lens = [0] * 70 + [5] + [0] * 5000 + [3, 0, 90] + [1] * 300 + [0] * 64 + [20]
    q, k, v, dout, cu = make(cuda, F16, 2, 1, 64, lens, pad=3, seed=20)
    check(run(q, k, v, dout, cu, max_len=90), q, k, v, dout, cu)


@pytest.mark.parametrize("window", [0, 700])
def test_shares_and_tiles_agree(cuda, window):
    """A wrong `max_len` changes how the work is cut (few long tiles, or each its own): the same sums in
    another order."""
    q, k, v, dout, cu = make(cuda, BF16, 8, 2, 64, (2000, 64, 64), seed=21)
    for n in (64, 2000):
        check(run(q, k, v, dout, cu, max_len=n, window=window), q, k, v, dout, cu, window=window)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lens, window", [((70,), 0), ((700, 40), 0), ((900,), 130)])
def test_values_of_unequal_size(cuda, dtype, lens, window):
    """Keys whose v is small or 0 beside others' (dS is as large as the others make it)."""
    q, k, v, dout, cu = make(cuda, dtype, 4, 2, 64, lens, seed=22, qscale=0.5, gscale=8.0, layout="plain")
    small = torch.arange(sum(lens)) % 3
    v[small == 0] *= 2.0 ** -12
    v[small == 1] = 0.0
    v[small == 2] *= 8.0
    dout[100:] *= 2.0 ** -8
    check(run(q, k, v, dout, cu, window=window), q, k, v, dout, cu, window=window)
    v[: sum(lens) // 2] *= 2.0 ** -6  # (what one share of the work sees is small, and not what its rows see)
    check(run(q, k, v, dout, cu, window=window), q, k, v, dout, cu, window=window)


@pytest.mark.parametrize("dtype, window", [(BF16, 500), (F16, 129)])
def test_long_with_a_window(cuda, dtype, window):
    """70001 rows; a stretch of 2000 in the middle and the last ones as sequences of their own are the same
    for rows whose keys, and keys whose rows, lie in the stretch."""
    q, k, v, dout, cu = make(cuda, dtype, 2, 1, 64, (70001,), seed=23, layout="plain")
    got = run(q, k, v, dout, cu, window=window)
    for a, b in ((33000, 35000), (68001, 70001)):
        s = slice(a, b)
        want = ref.attention(q[s], k[s], v[s], [0, b - a], dout[s], window=window)
        hi = b - a if b == 70001 else 1000
        for name in ("out", "stats", "dq", "dk", "dv"):
            ref.assert_within(got[name][s][500:hi], tuple(t[500:hi] for t in want[name]), name)


def test_one_long_sequence(cuda):
    """40000 rows of one sequence: the last rows, and the last keys, by the formulas alone."""
    n, last = 40000, 70
    q, k, v, dout, cu = make(cuda, BF16, 1, 1, 128, (n,), seed=24, layout="plain")
    got = run(q, k, v, dout, cu)
    q64, k64, v64, do = (t.double().cpu()[:, 0] for t in (q, k, v, dout))
    s = q64[-last:] @ k64.t() * 128 ** -0.5
    rows = torch.arange(n - last, n)[:, None]
    s = s.masked_fill(torch.arange(n)[None] > rows, -math.inf)
    p = torch.softmax(s, -1)
    o = p @ v64
    # a probability's error as in train_ref: a score's (twice), 8 half steps, and n of the sum
    es = (q64[-last:].abs() @ k64.abs().t()).amax(-1, keepdim=True) * 128 ** -0.5 * 136 * ref.U32
    half, ep = ref.HALF[BF16], 2 * es + (8 + n) * ref.U32
    oa = p @ v64.abs()
    off = (got["out"][-last:, 0].double().cpu() - o).abs()
    eo = half * o.abs() + (half + ep + n * ref.U32) * oa
    assert (off <= 1.01 * eo).all()
    # dS = P (dP - D): P's error of all, dP's and D's own (D's by the saved output's, too)
    dp, d = do[-last:] @ v64.t(), (do[-last:] * o).sum(-1, keepdim=True)
    ed = 136 * ref.U32 * (do[-last:].abs() @ v64.abs().t()) + (do[-last:].abs() * (1.01 * eo)).sum(-1, keepdim=True) \
        + 136 * ref.U32 * (do[-last:].abs() * o.abs()).sum(-1, keepdim=True)
    ds = p * (dp - d)
    eds = (ep + half) * ds.abs() + p * ed
    dq = ds @ k64 * 128 ** -0.5
    edq = 128 ** -0.5 * ((eds + n * ref.U32 * ds.abs()) @ k64.abs()) + half * dq.abs()
    assert ((got["dq"][-last:, 0].double().cpu() - dq).abs() <= 1.02 * edq).all()
    sl = slice(n - last, n)  # keys that only the last rows see
    dk, dv = ds[:, sl].t() @ q64[-last:] * 128 ** -0.5, p[:, sl].t() @ do[-last:]
    edk = 128 ** -0.5 * ((eds + n * ref.U32 * ds.abs())[:, sl].t() @ q64[-last:].abs()) + half * dk.abs()
    edv = ((half + ep + n * ref.U32) * p)[:, sl].t() @ do[-last:].abs() + half * dv.abs()
    assert ((got["dk"][-last:, 0].double().cpu() - dk).abs() <= 1.02 * edk).all()
    assert ((got["dv"][-last:, 0].double().cpu() - dv).abs() <= 1.02 * edv).all()


@pytest.mark.parametrize("heads, kv", [(40, 1), (40, 8), (9, 9), (66, 33)])
def test_head_groups(cuda, heads, kv):
    q, k, v, dout, cu = make(cuda, F16, heads, kv, 64, (130, 20), seed=25)
    check(run(q, k, v, dout, cu), q, k, v, dout, cu)


def test_strides_of_views(cuda):
    """Key heads that are one tensor's, expanded (a stride of 0), and gradients that come transposed."""
    from solution.layer import attention

    q, k, v, dout, cu = make(cuda, BF16, 4, 1, 64, (150, 9), seed=26, layout="plain")
    k4, v4 = k.expand(-1, 4, -1), v.expand(-1, 4, -1)
    check(run(q, k4, v4, dout, cu), q, k4, v4, dout, cu)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    out = attention(leaves[0], leaves[1].expand(-1, 4, -1), leaves[2].expand(-1, 4, -1), c)
    out.transpose(1, 2).backward(dout.transpose(1, 2).contiguous())
    got = run(q, k4, v4, dout, cu)
    assert torch.equal(leaves[0].grad, got["dq"])
    for x, name in zip(leaves[1:], ("dk", "dv")):  # (the sum over the expanded heads is autograd's)
        want = got[name].double().sum(1, keepdim=True)
        assert ((x.grad.double() - want).abs() <= 4 * ref.HALF[BF16] * got[name].double().abs().sum(1, keepdim=True)).all()


@pytest.mark.parametrize("cu", [[5, 60, 100], [-7, 40, 130], [100, 100], [0, 50, 20, 90], [70, 10], [0, 1 << 30]])
@pytest.mark.parametrize("window", [0, 9])
def test_offsets_that_leave_rows_out_or_make_no_sense(cuda, cu, window):
    """Rows before the first sequence and offsets outside of the rows: rows of no sequence are 0.  Offsets that
    decrease: nothing is defined but that what lies around the gradients stays as it is."""
    q, k, v, dout, _ = make(cuda, F16, 4, 2, 64, (100,), seed=27, layout="plain")
    c = torch.tensor(cu, dtype=torch.int32, device=cuda)
    from solution import kernels

    out, stats = kernels.attention_fwd(q, k, v, c, window=window)
    around = [torch.full((104, *t.shape[1:]), 7.0, dtype=F16, device=cuda) for t in (q, k, v)]
    grads = kernels.attention_bwd(dout, q, k, v, out, stats, c, window=window, grads=[t[2:102] for t in around])
    assert all((t[:2] == 7).all() and (t[102:] == 7).all() for t in around)
    if all(a <= b for a, b in zip(cu, cu[1:])):
        inside = [min(max(x, 0), 100) for x in cu]
        want = ref.attention(q, k, v, inside, dout, window=window)
        for name, t in zip(("out", "stats", "dq", "dk", "dv"), (out, stats, *grads)):
            ref.assert_within(t, want[name], name)


def test_a_second_derivative_raises(cuda):
    from solution.layer import attention, rope_attention

    q, k, v, dout, cu = make(cuda, F16, 4, 2, 64, (20,), seed=28, layout="plain")
    q.requires_grad_()
    g, = torch.autograd.grad(attention(q, k, v), q, dout.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
    x = torch.cat([t.detach().flatten(1) for t in (q, k, v)], 1).requires_grad_()
    cos = sin = torch.ones(20, 64, device=cuda)
    g, = torch.autograd.grad(rope_attention(x, cos, sin, 4, 2), x, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
