"""The paged-cache operators against their definition in 64 bits (tests/paged_ref.py): append
with rotation, attention with windows and sinks, attention behind a shared prefix."""

import math

import pytest
import torch

from tests import paged_ref as ref
from tests.gpu_util import banner

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def _append_check(s, kernels, cache, cos, sin, cu):
    q = kernels.paged_append(s.qkv.to(s.dev), cos.to(s.dev), sin.to(s.dev), cache, cu_q=cu)
    return q, s.k, s.v


def _table(positions, dim):
    from solution import kernels

    return kernels.rope_table(positions, dim, 1e4, "cpu")


APPENDS = [  # dtype, heads, kv, dim, page, lens, new, layout
    (F16, 12, 2, 128, 16, [1], [1], "slot"),
    (BF16, 28, 4, 128, 32, [33, 1, 64, 100], [1, 1, 1, 1], "slot"),
    (F16, 14, 2, 64, 16, [40, 7, 0, 16], [40, 3, 0, 1], "head"),
    (BF16, 4, 4, 64, 1, [5, 9], [5, 2], "padded"),
    (F16, 3, 1, 128, 128, [130, 70], [70, 70], "padded"),
    (BF16, 8, 1, 64, 64, [1] * 70, [1] * 70, "head"),
]


@pytest.mark.parametrize("dtype,heads,kv,dim,page,lens,new,layout", APPENDS)
@pytest.mark.parametrize("ragged", [False, True])
def test_append(cuda, dtype, heads, kv, dim, page, lens, new, layout, ragged):
    """q, k and v after an append.  A rotated value is lo c - hi s: two products and a sum in
    fp32 (3 half steps of fp32 on terms of |lo| + |hi| at most), rounded once to the type; v is
    a copy and slots that no token takes keep their bits (NaN)."""
    from solution import kernels

    if not ragged and len(set(new)) > 1:
        pytest.skip("one count of new tokens only")
    banner("append", dtype, heads, kv, dim, page, lens, new, layout, ragged)
    s = ref.Setup(cuda, dtype, heads, kv, dim, page, lens, new, seed=1, layout=layout)
    cos, sin = _table(max(lens) + 3, dim)
    q_ref, k_ref, v_ref = ref.append(s, cos, sin)
    cache = s.cache(kernels)
    q, k, v = _append_check(s, kernels, cache, cos, sin, s.cu_d() if ragged else None)
    size = s.qkv.double().abs().max()
    for got, want in ((q, q_ref), (k, k_ref)):
        got = got.double().cpu()
        assert torch.equal(got.isnan(), want.isnan())
        bound = want.abs() * ref.EPS[dtype] + 8 * 2.0 ** -24 * size
        assert ((got - want).abs().nan_to_num() <= bound.nan_to_num()).all()
    assert torch.equal(v.double().cpu().nan_to_num(-77.0), v_ref.nan_to_num(-77.0))


def test_append_out_of_range(cuda):
    """Positions below zero or past the rotation table: a q of zeros, nothing kept.  Pages that
    are not there (-1, past the cache): q kept, k and v dropped.  Tokens past the last offset: a
    q of zeros."""
    from solution import kernels

    s = ref.Setup(cuda, F16, 4, 2, 64, 16, [2, 40, 48, 20], [4, 3, 3, 1], seed=2)
    s.table[2, 2] = -1
    s.table[3, 1] = 1 << 20
    cos, sin = _table(39, 64)  # position 39 is past it
    q_ref, k_ref, v_ref = ref.append(s, cos, sin)
    cache = s.cache(kernels)
    pad = torch.cat((s.qkv, torch.ones(5, s.qkv.shape[1], dtype=F16)))  # 5 tokens of no sequence
    banner("append out of range")
    q = kernels.paged_append(pad.to(cuda), cos.to(cuda), sin.to(cuda), cache, cu_q=s.cu_d())
    assert not q[-5:].any() and not q[:2].any()
    torch.testing.assert_close(q[:-5].double().cpu(), q_ref, rtol=2.0 ** -10, atol=1e-5)
    for got, want in ((s.k, k_ref), (s.v, v_ref)):
        torch.testing.assert_close(got.double().cpu(), want, rtol=2.0 ** -10, atol=1e-5,
                                   equal_nan=True)


ATTENTIONS = [  # dtype, heads, kv, dim, page, lens, new, window, sinks, layout
    (F16, 12, 2, 128, 16, [1], [1], 0, 0, "slot"),
    (F16, 12, 2, 128, 16, [419], [1], 0, 0, "slot"),
    (BF16, 28, 4, 128, 32, [33, 1, 64, 600, 0, 31], [1] * 6, 0, 0, "slot"),
    (F16, 14, 2, 64, 16, [40, 7, 0, 163], [40, 3, 0, 1], 0, 0, "head"),
    (BF16, 4, 4, 64, 1, [5, 90], [5, 2], 0, 0, "padded"),
    (BF16, 16, 1, 128, 8, [300, 17], [2, 2], 0, 0, "padded"),
    (F16, 3, 1, 128, 128, [330, 70], [70, 70], 0, 0, "head"),
    (BF16, 40, 1, 64, 64, [129, 260], [1, 1], 0, 0, "slot"),
    # windows and sinks: inside one tile, across many, sinks past the window, window of one
    (F16, 12, 2, 128, 16, [700, 90, 3], [1, 1, 1], 64, 4, "slot"),
    (BF16, 14, 2, 64, 32, [700, 333], [5, 5], 100, 70, "head"),
    (F16, 8, 4, 64, 16, [257, 512, 64], [64, 200, 64], 33, 1, "slot"),
    (BF16, 7, 1, 128, 64, [400], [150], 1, 0, "slot"),
    (F16, 6, 2, 64, 16, [300, 20], [90, 20], 1, 3, "padded"),
    (F16, 2, 2, 128, 16, [200], [200], 1000, 2, "slot"),
    # more new tokens than positions: the first see nothing
    (F16, 6, 3, 64, 16, [3, 0, 40], [9, 4, 1], 0, 0, "slot"),
    (BF16, 6, 1, 128, 16, [2, 70], [30, 70], 16, 1, "slot"),
]


def _run(kernels, s, cuda, window=0, sinks=0, shared=0, **kw):
    cache = s.cache(kernels)
    args = dict(window=window, sinks=sinks, lse=True, **kw)
    if shared:
        return kernels.shared_prefix_attention(s.q.to(cuda), cache, shared, **args)
    return kernels.paged_attention(s.q.to(cuda), cache, **args)


def _check(got, want, dtype):
    (o, l), (ro, rl, vmax) = got, want
    ref.close(o, ro, vmax, dtype)
    empty = rl == -math.inf
    assert torch.equal(l.cpu() == -math.inf, empty) and not o.cpu()[empty].any()
    # scores of a few tens in fp32, exp's and log's few fp32 steps
    torch.testing.assert_close(l.cpu().double()[~empty], rl[~empty], rtol=1e-5, atol=2e-5)


@pytest.mark.parametrize("dtype,heads,kv,dim,page,lens,new,window,sinks,layout", ATTENTIONS)
@pytest.mark.parametrize("hints", ["none", "exact", "low"])
def test_attention(cuda, dtype, heads, kv, dim, page, lens, new, window, sinks, layout, hints):
    """Every shape without the host's hints, with exact ones and with hints that are too low
    (which may cost time, never a result)."""
    from solution import kernels

    banner("attention", dtype, heads, kv, dim, page, lens, new, window, sinks, layout, hints)
    s = ref.Setup(cuda, dtype, heads, kv, dim, page, lens, new, seed=3, layout=layout,
                  extra_width=9)
    kw = {"none": {}, "exact": dict(max_q=max(new), max_len=max(max(lens), 1)),
          "low": dict(max_q=1, max_len=1)}[hints]
    cu = None if len(set(new)) == 1 and hints != "low" else s.cu_d()
    _check(_run(kernels, s, cuda, window, sinks, cu_q=cu, **kw),
           ref.attention(s, window, sinks), dtype)


SHARED = [  # dtype, heads, kv, dim, page, shared, own lengths, new, window, sinks
    (F16, 12, 2, 128, 16, 201, [3, 40, 1], [1, 1, 1], 0, 0),
    (BF16, 28, 4, 128, 32, 96, [1] * 11, [1] * 11, 0, 0),
    (BF16, 14, 2, 64, 16, 513, [9, 140], [4, 4], 0, 0),
    (F16, 4, 4, 64, 64, 130, [7, 300, 66, 5], [1, 60, 3, 5], 0, 0),
    (F16, 12, 2, 128, 16, 330, [3, 40, 1], [1, 1, 1], 100, 4),   # windows reach into the prefix
    (BF16, 8, 1, 64, 16, 330, [30, 4], [1, 1], 16, 0),           # and miss it
    (F16, 8, 1, 64, 16, 330, [30, 4], [1, 1], 16, 340),          # sinks past it
    (BF16, 16, 1, 128, 16, 5, [2] * 9, [2] * 9, 0, 0),           # shorter than a page
    (F16, 12, 2, 128, 16, 64, [-1, 3, -64], [1, 1, 1], 0, 0),    # some end inside it, one empty
]


@pytest.mark.parametrize("dtype,heads,kv,dim,page,shared,tails,new,window,sinks", SHARED)
@pytest.mark.parametrize("hints", ["none", "exact"])
def test_shared_prefix(cuda, dtype, heads, kv, dim, page, shared, tails, new, window, sinks, hints):
    from solution import kernels

    banner("shared", dtype, heads, kv, dim, page, shared, tails, new, window, sinks, hints)
    lens = [shared + t for t in tails]
    s = ref.Setup(cuda, dtype, heads, kv, dim, page, lens, new, seed=4, shared=shared)
    kw = {} if hints == "none" else dict(max_q=max(new), max_len=max(lens))
    cu = None if len(set(new)) == 1 else s.cu_d()
    _check(_run(kernels, s, cuda, window, sinks, shared, cu_q=cu, **kw),
           ref.attention(s, window, sinks, shared), dtype)


def test_attention_pages_not_there(cuda):
    """Keys whose table entry names no page (-1, past the cache) are not seen, whatever lies
    behind; a sequence with no page at all gives zeros; so do tokens past the last offset."""
    from solution import kernels

    s = ref.Setup(cuda, F16, 8, 2, 64, 16, [200, 90, 60], [1, 3, 2], seed=5)
    s.table[0, 3:7] = -1
    s.table[1, 0] = 1 << 24
    s.table[2, :] = -5
    pad = torch.cat((s.q, torch.ones(7, 8, 64, dtype=F16)))
    banner("pages not there")
    want = ref.attention(s)
    cache = s.cache(kernels)
    for kw in ({}, dict(max_q=3, max_len=200)):
        o, l = kernels.paged_attention(pad.to(cuda), cache, cu_q=s.cu_d(), lse=True, **kw)
        _check((o[:-7], l[:-7]), want, F16)
        assert not o[-7:].any() and (l[-7:] == -math.inf).all()


@pytest.mark.parametrize("lens,new", [([90, 33], [1, 1]), ([90, 60], [60, 40])])
def test_attention_hidden_values_do_not_matter(cuda, lens, new):
    """Infinities and NaN in keys and values that a row does not see (past the window, behind a
    later token) leave that row alone."""
    from solution import kernels

    banner("hidden values", lens, new)
    s = ref.Setup(cuda, BF16, 4, 2, 64, 16, lens, new, seed=6)
    want = ref.attention(s, window=20, sinks=2)
    for b, (n, total) in enumerate(zip(new, lens)):
        j = total - n - 25 if n == 1 else total - 5  # hidden from all; from all but the last 5
        for x, bad in ((s.k, math.nan), (s.v, math.inf)):
            x[int(s.table[b, j // 16]), j % 16] = bad
            x[int(s.table[b, j // 16]), j % 16, 0, 3] = math.nan
    o, l = _run(kernels, s, cuda, 20, 2, cu_q=s.cu_d())
    rows = [t for b, n in enumerate(new) for t in range(s.starts[b], s.starts[b + 1])
            if n == 1 or t < s.starts[b + 1] - 5]
    _check((o[rows], l[rows]), tuple(x[rows] for x in want), BF16)


def test_attention_large_scores(cuda):
    """Scores of +-1e4: the running maximum keeps the exponentials in range, and the largest key
    decides alone."""
    from solution import kernels

    banner("large scores")
    s = ref.Setup(cuda, BF16, 4, 1, 128, 16, [300, 40], [1, 40], seed=7, qscale=2.0)
    s.q = torch.randn(41, 4, 128, generator=torch.Generator().manual_seed(8)).mul(2e3).to(BF16)
    ro, rl, vmax = ref.attention(s)
    o, l = _run(kernels, s, cuda, cu_q=s.cu_d())
    assert torch.isfinite(o.float()).all()
    torch.testing.assert_close(l.cpu().double(), rl, rtol=1e-5, atol=1e-3)
    # a score is off by up to 1e-6 of 1e4 in fp32, its exponential by 1e-2
    assert ((o.double().cpu() - ro).abs() <= (2.0 ** -7 + 2e-2) * vmax[..., None]).all()


def test_attention_strided_query(cuda):
    """q as the leading columns of a wider projection."""
    from solution import kernels

    banner("strided q")
    s = ref.Setup(cuda, F16, 6, 2, 64, 16, [50, 70], [2, 2], seed=9)
    wide = torch.full((4, 6 * 64 + 40), math.nan, dtype=F16)
    wide[:, 8:8 + 6 * 64] = s.q.view(4, -1)
    q = wide.to(cuda)[:, 8:8 + 6 * 64].unflatten(1, (6, 64))
    o, l = kernels.paged_attention(q, s.cache(kernels), lse=True)
    _check((o, l), ref.attention(s), F16)


def test_far_pages(cuda):
    """A cache whose last pages lie past 2^32 bytes (and 2^31 elements) of its first."""
    from solution import kernels

    banner("far pages")
    dim, kv, page = 64, 2, 16
    per = page * kv * dim
    pages = (1 << 31) // per + 300
    k = torch.empty((pages, page, kv, dim), dtype=F16, device=cuda)
    v = torch.empty_like(k)
    s = ref.Setup(cuda, F16, 4, kv, dim, page, [200, 45], [2, 2], seed=10)
    far = s.table.clone()
    far[far >= 0] += pages - s.k.shape[0]
    k[-s.k.shape[0]:], v[-s.k.shape[0]:] = s.k, s.v
    want = ref.attention(s)
    cos, sin = _table(256, dim)
    q_ref, k_ref, _ = ref.append(s, cos, sin)
    cache = kernels.PagedKV(k, v, far.to(cuda), torch.tensor(s.lens, dtype=torch.int32, device=cuda))
    _check(kernels.paged_attention(s.q.to(cuda), cache, lse=True), want, F16)
    kernels.paged_append(s.qkv.to(cuda), cos.to(cuda), sin.to(cuda), cache)
    torch.testing.assert_close(k[-s.k.shape[0]:].double().cpu(), k_ref, rtol=2.0 ** -10, atol=1e-5,
                               equal_nan=True)


def test_append_then_attend_in_a_graph(cuda):
    """Append and attention captured once and replayed with lengths that grow in place, eager
    work between the replays; every replay matches the eager calls bit for bit."""
    from solution import kernels

    banner("graph")
    s = ref.Setup(cuda, BF16, 12, 2, 128, 16, [700, 90, 5], [1, 1, 1], seed=11, extra_width=20)
    cos, sin = (t.to(cuda) for t in _table(2000, 128))
    s.table[:] = torch.randperm(s.table.numel()).view(s.table.shape).int()
    k = torch.randn(s.table.numel(), 16, 2, 128, device=cuda).to(BF16)
    v = torch.randn_like(k)
    lens = torch.tensor(s.lens, dtype=torch.int32, device=cuda)
    cache = kernels.PagedKV(k, v, s.table.to(cuda), lens)
    qkv = s.qkv.to(cuda)

    def step():
        q = kernels.paged_append(qkv, cos, sin, cache)
        return (kernels.paged_attention(q, cache, window=256, sinks=4),
                kernels.shared_prefix_attention(q, cache, 32))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for grow in (0, 1, 37, 150):
        lens += grow
        qkv.copy_(torch.randn_like(qkv.float()).to(BF16))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_other_stream_and_repeat(cuda):
    """On a stream of the caller's, twice: the same bits."""
    from solution import kernels

    banner("stream")
    s = ref.Setup(cuda, F16, 28, 4, 128, 16, [900, 30], [1, 1], seed=12)
    cache, q = s.cache(kernels), s.q.to(cuda)
    first = kernels.paged_attention(q, cache)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = kernels.paged_attention(q, cache)
    stream.synchronize()
    assert torch.equal(first, again)


# ---- many sequences, long tables, layouts that need 64-bit addresses

@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shared", [0, 40])
def test_many_ragged_sequences(cuda, ragged, shared):
    """More than two chunks of 64 sequences, of 0 to 1300 positions, cut into equal shares."""
    from solution import kernels

    banner("many sequences", ragged, shared)
    g = torch.Generator().manual_seed(20)
    lens = [shared + int(n) for n in torch.randint(0, 40, (131,), generator=g)]
    lens[5], lens[70], lens[130], lens[64] = shared + 1300, shared + 700, shared + 333, shared
    new = [1] * 131
    if ragged:
        for b in (0, 63, 64, 100):
            new[b] = b % 3  # some bring nothing, one two tokens
    s = ref.Setup(cuda, BF16, 4, 2, 64, 16, lens, new, seed=21, shared=shared)
    kw = dict(max_q=max(new), max_len=max(lens)) if ragged else {}
    _check(_run(kernels, s, cuda, shared=shared, cu_q=s.cu_d() if ragged else None, **kw),
           ref.attention(s, shared=shared), BF16)


@pytest.mark.parametrize("new,page", [(1, 16), (40, 16), (40, 8), (3, 32)])
def test_table_of_many_pages(cuda, new, page):
    """Lengths of several windows of 64 table entries, some entries missing, with and without a
    window of keys that starts far behind the sinks."""
    from solution import kernels

    banner("many pages", new, page)
    s = ref.Setup(cuda, F16, 2, 1, 64, page, [4100], [new], seed=22)
    s.table[0, 70], s.table[0, 100:103] = -1, 1 << 22
    for window, sinks in ((0, 0), (1500, 5)):
        _check(_run(kernels, s, cuda, window, sinks, cu_q=s.cu_d(), max_q=new, max_len=4100),
               ref.attention(s, window, sinks), F16)


@pytest.mark.parametrize("new", [1, 40])
def test_slots_far_apart(cuda, new):
    """Slot-major caches: a page's slots lie further apart than 32-bit byte offsets reach."""
    from solution import kernels

    banner("slots far apart", new)
    pages, page, kv, dim = 72000, 64, 4, 64
    k = torch.empty((page, pages, kv, dim), dtype=F16, device=cuda).transpose(0, 1)
    v = torch.empty((page, pages, kv, dim), dtype=F16, device=cuda).transpose(0, 1)
    s = ref.Setup(cuda, F16, 8, kv, dim, page, [300, 90], [new, new], seed=23)
    far = s.table.clone()
    far[far >= 0] += pages - s.k.shape[0]
    k[-s.k.shape[0]:], v[-s.k.shape[0]:] = s.k, s.v
    cache = kernels.PagedKV(k, v, far.to(cuda), torch.tensor(s.lens, dtype=torch.int32, device=cuda))
    _check(kernels.paged_attention(s.q.to(cuda), cache, lse=True), ref.attention(s), F16)


def test_values_not_finite_that_some_rows_see(cuda):
    """An infinity or NaN among the values reaches the rows that see its key, in that channel, and
    no other row; few rows and many."""
    from solution import kernels

    for new in (3, 40):
        banner("values not finite", new)
        s = ref.Setup(cuda, F16, 4, 2, 64, 16, [100], [new], seed=24)
        want = ref.attention(s)
        j = 100 - new // 2 - 1  # a position in the middle of the new tokens
        s.v[int(s.table[0, j // 16]), j % 16, 1, 7] = math.inf
        o, l = _run(kernels, s, cuda)
        p = torch.arange(100 - new, 100)
        hit = torch.zeros(o.shape, dtype=torch.bool)
        hit[p >= j, 2:, 7] = True
        assert (o.cpu()[hit] == math.inf).all()
        o = torch.where(hit.to(cuda), torch.zeros_like(o), o)
        want[0][hit] = 0
        _check((o, l), want, F16)


def test_queries_that_are_nan(cuda):
    """A query of NaN gives NaN (not the zeros of a query that sees nothing), pieces or not."""
    from solution import kernels

    for lens, new, shared in (([90], 1, 0), ([3000, 40], 1, 0), ([300], 40, 0), ([200, 190], 1, 150)):
        banner("NaN queries", lens, new, shared)
        s = ref.Setup(cuda, BF16, 4, 2, 64, 16, lens, [new] * len(lens), seed=25, shared=shared)
        want = ref.attention(s, shared=shared)
        s.q[-1, 1] = math.nan
        o, l = _run(kernels, s, cuda, shared=shared)
        assert o[-1, 1].isnan().all() and l[-1, 1].isnan()
        o[-1, 1], l[-1, 1] = want[0][-1, 1].to(o), want[1][-1, 1].to(l)
        _check((o, l), want, BF16)


def test_strides_of_single_rows(cuda):
    """A dimension of size one may have any stride: one token cut out of rows of an odd width, one
    page, one key/value head."""
    from solution import kernels

    banner("single rows")
    s = ref.Setup(cuda, F16, 2, 1, 64, 16, [11], [1], seed=26)
    wide = torch.full((2, 2 * 64 + 9), math.nan, dtype=F16, device=cuda)
    wide[0, :128] = s.q.view(-1).to(cuda)
    page = int(s.table[0, 0])
    k, v = (torch.as_strided(x[page].contiguous(), (1, 16, 1, 64), (n, 64, n, 1))
            for x, n in ((s.k, 5), (s.v, 3)))
    cache = kernels.PagedKV(k, v, torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                            torch.tensor([11], dtype=torch.int32, device=cuda))
    q = torch.as_strided(wide, (1, 2, 64), (137, 64, 1))
    _check(kernels.paged_attention(q, cache, lse=True), ref.attention(s), F16)


def test_refusals(cuda):
    """What the calls refuse, before any launch."""
    from solution import _lib, kernels

    s = ref.Setup(cuda, F16, 4, 2, 64, 16, [20], [1], seed=27)
    cache, q = s.cache(kernels), s.q.to(cuda)
    cos, sin = (t.to(cuda) for t in _table(32, 64))
    qkv = s.qkv.to(cuda)
    bad_calls = [
        lambda: kernels.paged_attention(s.q, cache),                          # host memory
        lambda: kernels.paged_attention(q.float(), cache),
        lambda: kernels.paged_attention(q[:, :3], cache),                     # heads % n_kv
        lambda: kernels.paged_attention(q[..., :32], cache),
        lambda: kernels.paged_attention(q, cache, cu_q=s.cu),                 # host offsets
        lambda: kernels.paged_attention(q, cache, cu_q=s.cu_d().long()),
        lambda: kernels.paged_attention(q, cache, out=torch.empty_like(q)[:, :2]),
        lambda: kernels.paged_append(s.qkv, cos, sin, cache),
        lambda: kernels.paged_append(qkv[:, :-64], cos, sin, cache),
        lambda: kernels.paged_append(qkv, cos[:, :16], sin, cache),
        lambda: kernels.paged_append(qkv, cos.double(), sin, cache),
        lambda: kernels.PagedKV(s.k, s.v[..., :32], cache.table, cache.lens),
        lambda: kernels.PagedKV(s.k, s.v, cache.table.long(), cache.lens),
        lambda: kernels.PagedKV(s.k, s.v, cache.table, cache.lens.cpu()),
    ]
    for call in bad_calls:
        with pytest.raises(ValueError):
            call()
    for kw in (dict(window=-1), dict(sinks=-1), dict(max_len=-1)):
        with pytest.raises(_lib.NF4LibraryError):
            kernels.paged_attention(q, cache, **kw)
    with pytest.raises(_lib.NF4Unsupported):  # rows of an odd width
        wide = torch.zeros(2, 4 * 64 + 3, dtype=F16, device=cuda)
        kernels.paged_attention(wide[:, :256].unflatten(1, (4, 64)), kernels.PagedKV(
            s.k, s.v, cache.table.repeat(2, 1), cache.lens.repeat(2)))


@pytest.mark.parametrize("heads,kv,new", [(7, 1, 5), (12, 1, 4), (6, 1, 7)])
@pytest.mark.parametrize("dim", [64, 128])
def test_three_row_blocks(cuda, heads, kv, new, dim):
    """33 to 48 rows a sequence over tables long enough for the kernel of few rows, ragged, with a
    window and without."""
    from solution import kernels

    banner("three row blocks", heads, kv, new, dim)
    s = ref.Setup(cuda, F16, heads, kv, dim, 16, [700, 90, new, 300], [new] * 4, seed=28,
                  extra_width=300)
    for window, sinks in ((0, 0), (4200, 3)):
        _check(_run(kernels, s, cuda, window, sinks), ref.attention(s, window, sinks), F16)
